"""Performance cases of products in 8-bit integers and of scores of given tokens: rows coded in 8 bits with a scale each, products of such rows, log
probabilities straight from a head's product without its logits, and log probabilities, ranks, entropies and top alternatives from logits.

Each operator has a plain form (elementary torch operations in 32 bits) and its call in the kernel-level C ABI (include/helix_b200_kernels.h).  Sizes are
those of this repository's configurations (helix_b200/configs.py: the 8B, 1B and 2B decoders).

A row of 8-bit codes c in -127..127 with a scale s stands for s c; s is the row's largest magnitude / 127 in fp32, c the whole number nearest to x / s, of two equally near
ones the even one.  Tokens are such rows of the left operand, channels such rows of the weights.
"""
import math

import torch

own = False
BF = torch.bfloat16


def listed():
    return [
        # the rows of a decode step, on their way into a projection: latency
        dict(name="rows_tokens", kind="rows", t=32, k=4096, f32=False),
        # the rows of a prompt step
        dict(name="rows_prompt", kind="rows", t=16001, k=4096, f32=False),
        # a checkpoint's down projections in fp32, coded when a model is loaded
        dict(name="rows_weights", kind="rows", t=4096, k=14336, f32=True),
        # one chat alone through the output projection
        dict(name="product_token", kind="product", m=1, n=4096, k=4096, epi="none"),
        # a chat batch through the gate and up projections
        dict(name="product_batch", kind="product", m=32, n=28672, k=4096, epi="swiglu"),
        # chunks of documents through a smaller model's first projection
        dict(name="product_odd", kind="product", m=777, n=8960, k=1536, epi="bias_gelu"),
        # a step of prompts through the gate and up projections
        dict(name="product_prompt", kind="product", m=8192, n=28672, k=4096, epi="swiglu"),
        # the next token of 32 running sequences: what the sampled ones cost
        dict(name="head_tokens", kind="head", t=32, v=128256, h=4096, q8=False, softcap=0.0),
        # a prompt of 2048 tokens scored (perplexity, reranking)
        dict(name="head_prompt", kind="head", t=2048, v=128256, h=4096, q8=False, softcap=0.0),
        # a shorter one by a model held in 8 bits, logits capped
        dict(name="head_codes", kind="head", t=701, v=151936, h=1536, q8=True, softcap=30.0),
        # logits of a step of sequences whose answers are bound to a grammar (nine tokens in ten are masked)
        dict(name="scores_step", kind="scores", t=32, v=128256, f32=True, masked=True, top=20),
        # logits of a whole prompt, in 16 bits to save their room
        dict(name="scores_prompt", kind="scores", t=2047, v=128256, f32=False, masked=False, top=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "product", "product", "product", "head", "head", "scores", "scores"])
    if kind == "rows":
        k = rng.choice([1536, 2048, 4096, 14336, _log_int(rng, 1, 15000)])
        return dict(kind="rows", t=_log_int(rng, 1, min(65000, 16001 * 4096 // k)), k=k, f32=rng.random() < 0.3)
    if kind == "product":
        n, k = rng.choice([(4096, 4096), (6144, 4096), (4096, 14336), (28672, 4096), (2048, 2048), (2048, 8192), (1536, 8960), (_log_int(rng, 1, 9000), _log_int(rng, 1, 9000))])
        epi = rng.choice(["none", "bias", "bias_gelu", "resid", "bias_resid", "swiglu", "f32"])
        if epi == "swiglu":
            n = -(-n // 256) * 256
        return dict(kind="product", m=rng.choice([_log_int(rng, 1, 64), _log_int(rng, 1, 8192)]), n=n, k=k, epi=epi)
    if kind == "head":
        v, h = rng.choice([(128256, 4096), (128256, 2048), (151936, 1536), (32768, 2048), (30522, 768), (_log_int(rng, 2, 150000), 8 * _log_int(rng, 1, 512))])
        return dict(kind="head", t=_log_int(rng, 1, 2048), v=v, h=h, q8=rng.random() < 0.4, softcap=rng.choice([0.0, 0.0, 30.0]))
    v = rng.choice([128256, 151936, 32768, 30522, _log_int(rng, 70, 152000)])
    return dict(kind="scores", t=_log_int(rng, 1, 2047 * 128256 // 152000), v=v, f32=rng.random() < 0.6, masked=rng.random() < 0.3,
                top=rng.choice([0, 1, 5, 20, rng.randint(2, 64)]))


# ------------------------------------------------------------------ inputs
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt * 7919) & 0x7FFFFFFF)


def _randn(seed, salt, shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=_gen(seed, salt), device="cuda", dtype=torch.float32) * scale).to(dtype)


def _up(n, to):
    return -(-n // to) * to


def _quantise(x):
    """Rows [.., K] -> codes (fp32 whole numbers) and scales [.., 1]; quotients in 64 bits, as many lie next to the middle of two codes."""
    top = x.abs().amax(-1, keepdim=True).float()
    s = top / torch.full_like(top, 127.0)
    c = torch.where(s > 0, (x.double() / s.double()).round(), torch.zeros((), dtype=torch.float64, device=x.device))
    return c.float(), s


def _code_rows(seed, salt, rows, k, scale):
    """Random rows as codes in rows of a multiple of 16 bytes, and their scales."""
    codes = torch.zeros(rows, _up(k, 16), dtype=torch.int8, device="cuda")
    scales = torch.zeros(rows, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // k)
    for i in range(0, rows, step):
        n = min(step, rows - i)
        c, s = _quantise(_randn(seed, salt + 31 * i, (n, k), scale, torch.float32))
        codes[i:i + n, :k], scales[i:i + n] = c.to(torch.int8), s[:, 0]
    return codes, scales


def _prepare_rows(case, seed):
    t, k = case["t"], case["k"]
    x = _randn(seed, 1, (t, k), 1.0, torch.float32)
    x *= 1 + 7 * (torch.arange(k, device="cuda") % 61 == 3)  # channels that stand out, as activations have them
    x = x.to(torch.float32 if case["f32"] else BF)
    if k % 8:  # rows that begin on 16 bytes
        x = torch.nn.functional.pad(x, (0, _up(k, 8) - k))[:, :k]
    ld = _up(k, 16)
    return dict(kind="rows", x=x, codes=torch.zeros(t, ld, dtype=torch.int8, device="cuda"), scales=torch.zeros(t, device="cuda"),
                seen=torch.zeros(t, ld, dtype=BF, device="cuda"), t=t, k=k, f32=case["f32"])


def _prepare_product(case, seed):
    m, n, k, epi = case["m"], case["n"], case["k"], case["epi"]
    wide = n // 2 if epi == "swiglu" else n
    x, xs = _code_rows(seed, 2, m, k, 1.0)
    w, ws = _code_rows(seed, 3, n, k, k ** -0.5)
    ld = _up(wide, 8)
    out = torch.zeros(m, ld, dtype=torch.float32 if epi == "f32" else BF, device="cuda")
    return dict(kind="product", x=x, xs=xs, w=w, ws=ws, bias=_randn(seed, 4, (n,)) if "bias" in epi else None, r=_randn(seed, 5, (m, ld)) if "resid" in epi else None,
                out=out, m=m, n=n, k=k, wide=wide, epi=epi)


def _prepare_head(case, seed):
    t, v, h = case["t"], case["v"], case["h"]
    if case["q8"]:
        (x, xs), (w, ws) = _code_rows(seed, 6, t, h, 1.0), _code_rows(seed, 7, v, h, 2.5 * h ** -0.5)
    else:
        x, xs, w, ws = _randn(seed, 6, (t, h)), None, _randn(seed, 7, (v, h), 2.5 * h ** -0.5), None
    return dict(kind="head", x=x, xs=xs, w=w, ws=ws, targets=torch.randint(0, v, (t,), generator=_gen(seed, 8), device="cuda").int(), lp=torch.zeros(t, device="cuda"),
                entropy=torch.zeros(t, device="cuda"), work=None, t=t, v=v, h=h, softcap=case["softcap"])


def _prepare_scores(case, seed):
    t, v, top = case["t"], case["v"], case["top"]
    top = min(top, v // 20 if case["masked"] else v)
    ld = _up(v, 8)
    x = torch.empty(t, ld, dtype=torch.float32 if case["f32"] else BF, device="cuda")
    targets = torch.randint(0, v, (t,), generator=_gen(seed, 9), device="cuda")
    step = max(1, (1 << 27) // v)
    for i in range(0, t, step):
        y = _randn(seed, 10 + 31 * i, (min(step, t - i), ld), 2.5, torch.float32)
        if case["masked"]:
            hide = torch.rand(y.shape, generator=_gen(seed, 11 + 31 * i), device="cuda") < 0.9
            hide.scatter_(1, targets[i:i + len(y), None], False)
            hide[:, :v // 20 * 10:10] = False  # (so that there are always some)
            y.masked_fill_(hide, -math.inf)
        x[i:i + len(y)] = y.to(x.dtype)
    return dict(kind="scores", x=x, targets=targets.int(), lp=torch.zeros(t, device="cuda"), entropy=torch.zeros(t, device="cuda"),
                rank=torch.zeros(t, dtype=torch.int32, device="cuda"), ids=torch.zeros(t, max(top, 1), dtype=torch.int32, device="cuda"),
                top_lp=torch.zeros(t, max(top, 1), device="cuda"), t=t, v=v, top=top, f32=case["f32"])


def prepare(case, seed):
    return {"rows": _prepare_rows, "product": _prepare_product, "head": _prepare_head, "scores": _prepare_scores}[case["kind"]](case, seed)


# ------------------------------------------------------------------ plain forms
def _plain_rows(s):
    c, d = _quantise(s["x"])
    return [(c * d).to(BF), d[:, 0]]


def _plain_product(s):
    y = s["x"][:, :s["k"]].float() @ s["w"][:, :s["k"]].float().T
    y *= s["ws"]
    y *= s["xs"][:, None]
    if s["bias"] is not None:
        y += s["bias"].float()
    if s["epi"] == "bias_gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    if s["epi"] == "swiglu":  # rows of the weights: 128 of the gate, 128 beside them, and so on
        g, u = y.unflatten(1, (-1, 2, 128)).unbind(2)
        y = (g / (1 + torch.exp(-g)) * u).flatten(1)
    if s["r"] is not None:
        y += s["r"][:, :s["n"]].float()
    return y.to(s["out"].dtype)


def _plain_softmax(x, targets):
    """Rows of fp32 logits -> log probability of the target, entropy, log of the sum of exponentials."""
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(-1)
    mean = torch.where(e > 0, e * d, 0).sum(-1) / total
    lse = top[:, 0] + torch.log(total)
    at = torch.gather(x, 1, targets.long()[:, None])[:, 0]
    return at - lse, torch.log(total) - mean, lse, at


def _plain_head(s):
    x, w = s["x"][:, :s["h"]].float(), s["w"][:, :s["h"]].float()
    y = x @ w.T
    if s["ws"] is not None:
        y *= s["ws"]
        y *= s["xs"][:, None]
    if s["softcap"] > 0:
        y = s["softcap"] * torch.tanh(y / s["softcap"])
    return list(_plain_softmax(y, s["targets"])[:2])


def _plain_scores(s):
    x = s["x"][:, :s["v"]].float()
    lp, entropy, lse, at = _plain_softmax(x, s["targets"])
    j = torch.arange(s["v"], device="cuda")
    before = (x > at[:, None]) | ((x == at[:, None]) & (j < s["targets"][:, None]))
    rank = before.sum(-1).int()
    val, ids = torch.sort(x + 0.0, dim=-1, descending=True, stable=True)
    return [lp, entropy, rank, ids[:, :s["top"]].int(), val[:, :s["top"]] - lse[:, None]]


# ------------------------------------------------------------------ the framework's calls
def _p(t):
    return None if t is None else t.data_ptr()


def _lib():
    from helix_b200 import lib
    return lib()


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"status {rc}: {_lib().hbk_last_error().decode()}")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_rows(s):
    _ok(_lib().hbk_rows_q8(_p(s["x"]), int(s["f32"]), s["x"].stride(0), _p(s["codes"]), s["codes"].stride(0), _p(s["scales"]), _p(s["seen"]), s["seen"].stride(0),
                           s["t"], s["k"], _stream()))
    return [s["seen"][:, :s["k"]], s["scales"]]


def _own_product(s):
    epi = {"none": 0, "bias": 1, "bias_gelu": 2, "resid": 3, "bias_resid": 4, "swiglu": 5, "f32": 6}[s["epi"]]
    ld = s["out"].stride(0)
    _ok(_lib().hbk_gemm_q8(_p(s["x"]), s["x"].stride(0), _p(s["xs"]), _p(s["w"]), s["w"].stride(0), _p(s["ws"]), _p(s["out"]), ld, _p(s["r"]), ld, _p(s["bias"]),
                           s["m"], s["n"], s["k"], epi, _stream()))
    return s["out"][:, :s["wide"]]


def _own_head(s):
    l = _lib()
    if s["work"] is None:
        s["work"] = torch.empty(l.hbk_head_scores_workspace_floats(s["t"], s["v"]), device="cuda", dtype=torch.float32)
    _ok(l.hbk_head_scores(_p(s["x"]), s["x"].stride(0), _p(s["xs"]), _p(s["w"]), s["w"].stride(0), _p(s["ws"]), _p(s["targets"]), _p(s["lp"]), _p(s["entropy"]),
                          _p(s["work"]), s["t"], s["v"], s["h"], 1.0, s["softcap"], _stream()))
    return [s["lp"], s["entropy"]]


def _own_scores(s):
    _ok(_lib().hbk_token_scores(_p(s["x"]), int(s["f32"]), s["x"].stride(0), _p(s["targets"]), s["t"], s["v"], s["top"], _p(s["lp"]), _p(s["rank"]), _p(s["entropy"]),
                                _p(s["ids"]), _p(s["top_lp"]), _stream()))
    return [s["lp"], s["entropy"], s["rank"], s["ids"][:, :s["top"]], s["top_lp"][:, :s["top"]]]


def run(state):
    kind = state["kind"]
    if own:
        return {"rows": _own_rows, "product": _own_product, "head": _own_head, "scores": _own_scores}[kind](state)
    return {"rows": _plain_rows, "product": _plain_product, "head": _plain_head, "scores": _plain_scores}[kind](state)


# ------------------------------------------------------------------ work and values in 64 bits
def work(case):
    if case["kind"] == "rows":
        n = case["t"] * case["k"]
        return dict(bytes=n * ((4 if case["f32"] else 2) + 1 + 2) + 4 * case["t"], flops=4 * n)
    if case["kind"] == "product":
        m, n, k, epi = (case[x] for x in ("m", "n", "k", "epi"))
        wide = n // 2 if epi == "swiglu" else n
        more = m * wide * 2 * ("resid" in epi) + n * 2 * ("bias" in epi)
        return dict(bytes=n * k + m * k + 4 * (m + n) + m * wide * (4 if epi == "f32" else 2) + more, flops=2 * m * n * k)
    if case["kind"] == "head":
        t, v, h = case["t"], case["v"], case["h"]
        return dict(bytes=(t + v) * (h + 4 if case["q8"] else 2 * h) + 12 * t, flops=2 * t * v * h)
    t, v = case["t"], case["v"]
    return dict(bytes=t * v * (4 if case["f32"] else 2) + t * (16 + 8 * case["top"]), flops=6 * t * v)


def _exact_scores(x, targets):
    """One row after the other's block of fp64 logits; a masked token has weight 0."""
    hi = x.max(-1).values
    p = (x - hi[:, None]).exp()
    z = p.sum(-1)
    lse = hi + z.log()
    p = p / z[:, None]
    entropy = -torch.special.xlogy(p, p).sum(-1)
    return x[torch.arange(len(x), device="cuda"), targets.long()] - lse, entropy, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rows":
        x = s["x"].double()
        d = (x.abs().max(-1).values / 127).float().double()
        return [torch.round(x / d[:, None]).nan_to_num(0.0) * d[:, None], x.abs().max(-1).values / 127]
    if case["kind"] == "product":
        k = s["k"]
        y = torch.mm(s["x"][:, :k].double() * s["xs"].double()[:, None], (s["w"][:, :k].double() * s["ws"].double()[:, None]).T)
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if case["epi"] == "bias_gelu":
            y = y * torch.special.ndtr(y)
        if case["epi"] == "swiglu":
            cols = torch.arange(s["wide"], device="cuda")
            gate = cols // 128 * 256 + cols % 128
            y = y[:, gate] * torch.sigmoid(y[:, gate]) * y[:, gate + 128]
        if s["r"] is not None:
            y = y + s["r"].double()[:, :s["n"]]
        return y
    if case["kind"] == "head":
        h = s["h"]
        w = s["w"][:, :h].double()
        if s["ws"] is not None:
            w *= s["ws"].double()[:, None]
        lp, entropy = [], []
        for i in range(0, s["t"], 512):
            x = s["x"][i:i + 512, :h].double()
            if s["xs"] is not None:
                x = x * s["xs"][i:i + 512].double()[:, None]
            y = x @ w.T
            if case["softcap"] > 0:
                y = torch.tanh(y / case["softcap"]) * case["softcap"]
            a, b, _ = _exact_scores(y, s["targets"][i:i + 512])
            lp.append(a)
            entropy.append(b)
        return [torch.cat(lp), torch.cat(entropy)]
    out = [[], [], [], [], []]
    for i in range(0, s["t"], 256):
        x, g = s["x"][i:i + 256, :s["v"]].double(), s["targets"][i:i + 256].long()
        lp, entropy, lse = _exact_scores(x, g)
        at = x.gather(1, g[:, None])
        rank = (x > at).sum(-1) + ((x == at).cumsum(-1) - 1).gather(1, g[:, None])[:, 0]
        left, ids, val = x.clone(), [], []
        for _ in range(s["top"]):  # the largest, the first of equals, again and again
            v = left.max(-1, keepdim=True).values
            j = (left == v).int().argmax(-1, keepdim=True)
            ids.append(j)
            val.append(v)
            left.scatter_(1, j, -math.inf)
        none = torch.zeros(len(x), 0, device="cuda")
        for o, y in zip(out, (lp, entropy, rank.int(), torch.cat(ids, 1).int() if ids else none.int(), torch.cat(val, 1) - lse[:, None] if val else none.double())):
            o.append(y)
    return [torch.cat(o) for o in out]
