"""Performance cases of a decode step whose cache and weights are held in 4 bits: page tables and slot maps made on the GPU, cache rows written in
4 bits, attention over them, and products with 4-bit weights.

Each operator has a plain form (elementary torch operations in 32 bits) and its call in the kernel-level C ABI
(include/helix_b200_kernels.h).  Sizes are those of this repository's configurations (helix_b200/configs.py: the 8B, 1B and 2B decoders).

The 4-bit format: 32 neighbouring entries share a scale d, a code c stands for d (c - 8).  A row of cache codes is laid out in words of eight
entries (keys) or in half words of four entries with the two positions of a pair side by side (values); a page of one kv head holds 64 rows of
codes, then 64 rows of scales.  Weights are tiles of 16 rows x 128 columns with the rows laid out as keys are.
"""
import math

import torch

own = False
BF = torch.bfloat16
PAGE = 64


def listed():
    return [
        # a decode step of a chat batch: every request gets one token, one in 64 of them a page, some have ended
        dict(name="tables_tokens", kind="tables", reqs=48, ctx=2048, longest_new=1, ended=5, pages=4096, max_pages=128),
        # a step of a busy server: many running sequences and new prompts, 16k rows in all
        dict(name="tables_prompts", kind="tables", reqs=700, ctx=8192, longest_new=160, ended=40, pages=100000, max_pages=200),
        # the rows of a decode step: 32 sequences, 8 kv heads
        dict(name="write_tokens", kind="write", rows=32, hkv=8, d=128, pages=1024),
        # the rows of a prompt step
        dict(name="write_prompts", kind="write", rows=16001, hkv=8, d=128, pages=512),
        # one chat alone on the GPU: latency
        dict(name="attn_one", kind="attn", seqs=1, shortest=777, longest=777, rows=1, hq=32, hkv=8, d=128, window=0, softcap=0.0, sink=False),
        # one decode step of 32 sequences with about 2k positions each
        dict(name="attn_tokens", kind="attn", seqs=32, shortest=1500, longest=2176, rows=1, hq=32, hkv=8, d=128, window=0, softcap=0.0, sink=False),
        # long contexts: few sequences, so the cache is split over the machine
        dict(name="attn_long", kind="attn", seqs=3, shortest=9000, longest=131000, rows=1, hq=32, hkv=8, d=128, window=0, softcap=0.0, sink=False),
        # heads of 64 entries with a window, capped scores and sinks, lengths from one position on
        dict(name="attn_window", kind="attn", seqs=96, shortest=1, longest=6000, rows=1, hq=32, hkv=8, d=64, window=4096, softcap=50.0, sink=True),
        # portions of prompts against everything cached before them
        dict(name="attn_portion", kind="attn", seqs=3, shortest=900, longest=5000, rows=97, hq=12, hkv=2, d=128, window=0, softcap=0.0, sink=False),
        # one token through the output projection
        dict(name="product_token", kind="product", m=1, n=4096, k=4096, epi="none"),
        # a chat batch through the down projection, added to the stream
        dict(name="product_down", kind="product", m=13, n=4096, k=14336, epi="resid"),
        # a batch through the gate and up projections
        dict(name="product_gate_up", kind="product", m=32, n=28672, k=4096, epi="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attn", "attn", "portion", "product", "product"])
    if kind == "tables":
        reqs = _log_int(rng, 1, 1000)
        return dict(kind="tables", reqs=reqs, ctx=_log_int(rng, 1, 8000), longest_new=rng.choice([1, 1, _log_int(rng, 2, 200)]), ended=rng.randint(0, reqs // 8),
                    pages=200000, max_pages=rng.randint(140, 260))
    if kind == "write":
        return dict(kind="write", rows=_log_int(rng, 1, 16000), hkv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128]), pages=rng.randint(256, 1024))
    hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 64), (12, 2, 128), (32, 32, 128), (8, 1, 128), (9, 3, 64)])
    if kind == "attn":
        seqs = _log_int(rng, 1, 128)
        longest = min(_log_int(rng, 1, 100000), 200000 * 8 // (seqs * hkv))
        return dict(kind="attn", seqs=seqs, shortest=rng.randint(1, longest), longest=longest, rows=1, hq=hq, hkv=hkv, d=d, window=rng.choice([0, 0, _log_int(rng, 1, 4096)]),
                    softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.choice([False, False, True]))
    if kind == "portion":
        rows = _log_int(rng, 2, 200)
        return dict(kind="attn", seqs=rng.randint(1, 3), shortest=rows, longest=rows + _log_int(rng, 1, 4500), rows=rows, hq=hq, hkv=min(hkv, 8) if hq != 32 or hkv != 32 else 8, d=d,
                    window=rng.choice([0, 0, _log_int(rng, 1, 2000)]), softcap=0.0, sink=rng.choice([False, True]))
    n, k = rng.choice([(4096, 4096), (6144, 4096), (4096, 14336), (28672, 4096), (2048, 2048), (2048, 8192), (1536, 8960), (_log_int(rng, 1, 9000), 32 * _log_int(rng, 1, 300))])
    return dict(kind="product", m=_log_int(rng, 1, 32), n=n, k=k, epi=rng.choice(["none", "bias", "resid", "bias_resid", "f32"]))


# ------------------------------------------------------------------ inputs
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt * 7919) & 0x7FFFFFFF)


def _randn(seed, salt, shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=_gen(seed, salt), device="cuda", dtype=torch.float32) * scale).to(dtype)


def _spread(n, lo, hi):
    """n unequal lengths between lo and hi: part of the case, not of the seed, so that every seed is the same work."""
    return [lo + (hi - lo) * ((i * 7 + 3) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _quantise(x, scale_type):
    """x [..., 32] fp32 -> codes (uint8) and the scale of each group, in fp32."""
    at = x.abs().argmax(-1, keepdim=True)
    m = torch.gather(x, -1, at)
    d = (m / -8).to(scale_type).float()
    c = torch.where(d == 0, torch.full_like(x, 8), torch.floor(x / d + 8.5).clamp(0, 15))
    return c.to(torch.uint8), d[..., 0]


def _key_bytes(c):
    """codes [..., 64 or 128] of a row -> its bytes: word j of quarter t holds entries 32 j + 8 t + i, i even in nibble i / 2, odd in nibble 4 + i / 2."""
    w = c.unflatten(-1, (-1, 4, 8)).transpose(-3, -2)  # [..., quarter, group, entry]
    w = w[..., [0, 2, 4, 6, 1, 3, 5, 7]]
    return (w[..., 0::2] | w[..., 1::2] << 4).flatten(-3)


def _key_codes(b):
    w = b.unflatten(-1, (4, -1, 4))
    w = torch.stack([w & 15, w >> 4], -1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    return w.transpose(-3, -2).flatten(-3)


def _value_order(d):
    """Chunk g of a pair of positions lies at place g ^ x of the pair's row."""
    pair = torch.arange(PAGE // 2, device="cuda")[:, None]
    return torch.arange(8, device="cuda")[None] ^ ((pair & 3) << 1 if d == 128 else (pair & 2) << 1)


def _value_bytes(c):
    """codes [..., 64 positions, D] of a page -> its bytes: [pair][place][group][position of the pair][two bytes of entries 32 j + 4 g + 0..3]."""
    d = c.shape[-1]
    w = c.unflatten(-1, (-1, 8, 4)).unflatten(-4, (-1, 2))  # [pair, half, group, chunk, entry]
    w = (w[..., 0::2] | w[..., 1::2] << 4).movedim(-2, -4)  # [pair, chunk, half, group, byte]
    w = w.transpose(-3, -2)
    at = _value_order(d)[..., None, None, None].expand(w.shape[-5:]).expand(w.shape)
    return torch.zeros_like(w).scatter_(-4, at, w).flatten(-5)


def _value_codes(b, d):
    w = b.unflatten(-1, (PAGE // 2, 8, d // 32, 2, 2))
    at = _value_order(d)[..., None, None, None].expand(w.shape[-5:]).expand(w.shape)
    w = torch.gather(w, -4, at).transpose(-3, -2).movedim(-4, -2)  # [pair, half, group, chunk, byte]
    return torch.stack([w & 15, w >> 4], -1).flatten(-2).flatten(-3).flatten(-3, -2)


def _page_bytes(c, s, keys):
    codes = _key_bytes(c).flatten(-2) if keys else _value_bytes(c)
    return torch.cat([codes, s.to(BF).contiguous().view(torch.uint8).flatten(-2)], -1)


def _page_values(b, d, keys):
    """Bytes of pages [..., block] -> fp32 [..., 64, D]."""
    n = PAGE * d // 2
    c = _key_codes(b[..., :n].unflatten(-1, (PAGE, -1))) if keys else _value_codes(b[..., :n], d)
    s = b[..., n:].contiguous().view(BF).unflatten(-1, (PAGE, -1)).float()
    return (c.unflatten(-1, (-1, 32)).float() - 8).mul_(s[..., None]).flatten(-2)


def _random_plane(seed, salt, pages, hkv, d, keys):
    plane = torch.empty(pages, hkv, PAGE * d // 2 + PAGE * d // 16, dtype=torch.uint8, device="cuda")
    step = 2048
    for i in range(0, pages, step):
        x = _randn(seed, salt + 31 * i, (min(step, pages - i), hkv, PAGE, d // 32, 32), dtype=torch.float32)
        c, s = _quantise(x, BF)
        plane[i:i + step] = _page_bytes(c.flatten(-2), s, keys)
    return plane


def _prepare_tables(case, seed):
    b = case["reqs"]
    g = _gen(seed, 1)
    ctx = torch.randint(0, case["ctx"] + 1, (b,), generator=g, device="cuda").int()
    new = torch.randint(1, case["longest_new"] + 1, (b,), generator=g, device="cuda").int()
    new[torch.randperm(b, generator=g, device="cuda")[:case["ended"]]] = -1
    held = (ctx + PAGE - 1) // PAGE
    ids = torch.randperm(case["pages"], generator=g, device="cuda").int()
    first = held.cumsum(0) - held
    at = torch.arange(case["max_pages"], device="cuda")[None]
    table = torch.where(at < held[:, None], ids[(first[:, None] + at).clamp(max=case["pages"] - 1)], -1).int()
    used = int(held.sum())
    free = torch.full((case["pages"],), -1, dtype=torch.int32, device="cuda")
    free[:case["pages"] - used] = ids[used:]
    t = b * case["longest_new"]
    out = dict(cu=_ints([0] * (b + 1)), kv=_ints([0] * b), pos=_ints([0] * t), slot=_ints([0] * t), left=_ints([0]))
    return dict(ctx=ctx, new=new, table=table, free=free, count=_ints([case["pages"] - used]), out=out, t=t, **{k: case[k] for k in ("kind", "pages", "max_pages")})


def _prepare_write(case, seed):
    t, hkv, d = case["rows"], case["hkv"], case["d"]
    kv = _randn(seed, 2, (t, 2, hkv, d))
    kv = (kv * (1 + 7 * (torch.arange(d, device="cuda") % 29 == 3))).to(BF)  # channels that stand out, as keys have them
    slots = torch.randperm(case["pages"], generator=_gen(seed, 3), device="cuda")
    if t <= 64:  # one token of each of many sequences
        slots = slots[:t] * PAGE + torch.randint(0, PAGE, (t,), generator=_gen(seed, 4), device="cuda")
    else:
        slots = (slots[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()[5:5 + t]
    planes = [torch.zeros(case["pages"], hkv, PAGE * d // 2 + PAGE * d // 16, dtype=torch.uint8, device="cuda") for _ in range(2)]
    seen = [torch.zeros(t, hkv, d, dtype=BF, device="cuda") for _ in range(2)]
    return dict(kv=kv, slots=slots.int(), planes=planes, seen=seen, **{k: case[k] for k in ("kind", "hkv", "d", "pages")}, t=slots.numel())


def _portions(case):
    lens = _spread(case["seqs"], case["shortest"], case["longest"])
    rows = [min(n, max(1, case["rows"] - 13 * i)) if case["rows"] > 1 else 1 for i, n in enumerate(lens)]
    return lens, rows


def _prepare_attn(case, seed):
    lens, rows = _portions(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    width = max(-(-n // PAGE) for n in lens)
    need = sum(-(-n // PAGE) for n in lens)
    ids = torch.randperm(need, generator=_gen(seed, 5), device="cuda").int()
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        p = -(-n // PAGE)
        table[b, :p] = ids[at:at + p]
        at += p
    t = sum(rows)
    first = [sum(rows[:b]) for b in range(len(rows))]
    # rows of the packed batch by sequence, the last row again where a portion is shorter
    at = _ints([[f + min(i, r - 1) for i in range(max(rows))] for f, r in zip(first, rows)]).long()
    mask = _ints([[i < r for i in range(max(rows))] for r in rows]).bool()
    state = dict(q=_randn(seed, 6, (t, hq, d), 1.5), k=_random_plane(seed, 7, need, hkv, d, True), v=_random_plane(seed, 8, need, hkv, d, False), table=table,
                 kv=_ints(lens), cu=_ints(first + [t]), at=at, mask=mask, rows=_ints(rows), sink=_randn(seed, 9, (hq,)) if case["sink"] else None,
                 out=torch.zeros(t, hq, d, dtype=BF, device="cuda"), t=t, most_rows=max(rows), longest=max(lens), width=width, pages=need, split=0,
                 scale=d ** -0.5, work=None, **{k: case[k] for k in ("kind", "seqs", "hq", "hkv", "d", "window", "softcap")})
    return state


def _prepare_product(case, seed):
    m, n, k = case["m"], case["n"], case["k"]
    nt, kt = -(-n // 16), -(-k // 128)
    codes = torch.full((nt * 16, kt * 128), 8, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(nt * 16, kt * 4, dtype=torch.float16, device="cuda")
    c, s = _quantise(_randn(seed, 10, (n, k // 32, 32), k ** -0.5, torch.float32), torch.float16)
    codes[:n, :k], scales[:n, :k // 32] = c.flatten(1), s.half()
    tiles = _key_bytes(codes.view(nt, 16, kt, 128).transpose(1, 2)).flatten(-2)
    sc = scales.view(nt, 16, kt, 4).transpose(1, 2).contiguous().view(torch.uint8).flatten(-2)
    out = torch.zeros(m, n, dtype=torch.float32 if case["epi"] == "f32" else BF, device="cuda")
    return dict(kind="product", x=_randn(seed, 11, (m, k)), w=torch.cat([tiles, sc], -1), bias=_randn(seed, 12, (n,)) if "bias" in case["epi"] else None,
                r=_randn(seed, 13, (m, n)) if "resid" in case["epi"] else None, out=out, m=m, n=n, k=k, epi=case["epi"])


def prepare(case, seed):
    return {"tables": _prepare_tables, "write": _prepare_write, "attn": _prepare_attn, "product": _prepare_product}[case["kind"]](case, seed)


# ------------------------------------------------------------------ plain forms
def _plain_tables(s):
    ctx, new, count, t, mp = s["ctx"].long(), s["new"].long(), s["count"].long()[0], s["t"], s["max_pages"]
    held = (ctx + PAGE - 1) // PAGE
    ended, n = new < 0, new.clamp(min=0)
    back = torch.where(ended, held, 0)
    back_end, row_end = back.cumsum(0), n.cumsum(0)
    after = (ctx + n + PAGE - 1) // PAGE
    fits = (after <= mp) & (row_end <= t)
    need = torch.where(fits & ~ended, after - held, 0)
    end = need.cumsum(0)
    top = count + back_end[-1]
    ok = fits & ((need == 0) | (end <= top))
    left = top - torch.where(ok & (need > 0), end, 0).max()

    def on_stack(i):
        j = (i - count).clamp(min=0)
        b = torch.searchsorted(back_end, j, right=True).clamp(max=len(ctx) - 1)
        page = s["table"][b, (j - (back_end - back)[b]).clamp(0, mp - 1)]
        return torch.where(i < count, s["free"][i.clamp(0, s["pages"] - 1)], page)

    row = torch.arange(t, device="cuda")
    b = torch.searchsorted(row_end, row, right=True)
    live, b = b < len(ctx), b.clamp(max=len(ctx) - 1)
    pos = ctx[b] + row - (row_end - n)[b]
    at = pos // PAGE - held[b]
    page = torch.where(at < 0, s["table"][b, (pos // PAGE).clamp(max=mp - 1)], on_stack(top - 1 - ((end - need)[b] + at.clamp(min=0))))
    slot = torch.where(live & ok[b], page * PAGE + pos % PAGE, -1)
    col = torch.arange(mp, device="cuda")[None] - held[:, None]
    taken = on_stack((top - 1 - (end - need)[:, None] - col.clamp(min=0)).clamp(min=0))
    table = torch.where((col >= 0) & (col < need[:, None]) & ok[:, None], taken, s["table"])
    i = torch.arange(s["pages"], device="cuda")
    free = torch.where((i >= count) & (i < left), on_stack(i), s["free"])
    cu = torch.cat([row_end.new_zeros(1), row_end.clamp(max=t)])
    kv = torch.where(ended, 0, torch.where(ok, ctx + n, ctx))
    return [x.int() for x in (table, free, left[None], cu, kv, torch.where(live, pos, 0), slot)]


def _plain_write(s):
    c, d = _quantise(s["kv"].float().unflatten(-1, (-1, 32)), BF)
    seen = ((c.float() - 8) * d[..., None]).flatten(-2).to(BF)
    return [seen[:, 0], seen[:, 1]]


def _plain_attn(s):
    b, hkv, d, group = s["seqs"], s["hkv"], s["d"], s["hq"] // s["hkv"]
    # [sequence, kv head, position, entry]
    k, v = (_page_values(s[x][s["table"].long()], d, x == "k").transpose(1, 2).flatten(2, 3) for x in ("k", "v"))
    q = s["q"].float()[s["at"]].unflatten(2, (hkv, group)).permute(0, 2, 1, 3, 4)  # [sequence, kv head, row, head, entry]
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (-1, group)) * s["scale"]
    if s["softcap"] > 0:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    j = torch.arange(k.shape[2], device="cuda")
    last = (s["kv"] - s["rows"])[:, None] + torch.arange(s["most_rows"], device="cuda")[None]
    sees = j <= last[..., None]
    if s["window"] > 0:
        sees = sees & (j > last[..., None] - s["window"])
    x = x.masked_fill(~sees[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sink"] is not None:
        extra = s["sink"].float().view(1, hkv, 1, group, 1)
        top = torch.maximum(top, extra)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(extra - top)
    o = torch.matmul((p / total).flatten(2, 3), v).unflatten(2, (-1, group))
    return o.permute(0, 2, 1, 3, 4).flatten(2, 3)[s["mask"]].to(BF)


def _plain_product(s):
    nt, kt = -(-s["n"] // 16), -(-s["k"] // 128)
    c = _key_codes(s["w"][..., :1024].unflatten(-1, (16, 64)))
    d = s["w"][..., 1024:].contiguous().view(torch.float16).unflatten(-1, (16, 4)).float()
    w = (c.unflatten(-1, (4, 32)).float() - 8) * d[..., None]
    w = w.flatten(-2).transpose(1, 2).reshape(nt * 16, kt * 128)[:s["n"], :s["k"]]
    y = s["x"].float() @ w.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["out"].dtype)


# ------------------------------------------------------------------ the framework's calls
def _p(t):
    return None if t is None else t.data_ptr()


def _lib():
    from helix_b200 import lib
    return lib()


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"status {rc}: {_lib().hbk_last_error().decode()}")


def _own_tables(s):
    o = s["out"]
    _ok(_lib().hbk_page_tables(_p(s["ctx"]), _p(s["new"]), s["ctx"].numel(), _p(s["table"]), s["max_pages"], _p(s["free"]), _p(s["count"]), _p(o["left"]), s["pages"],
                               _p(o["cu"]), _p(o["kv"]), _p(o["pos"]), _p(o["slot"]), s["t"], PAGE, torch.cuda.current_stream().cuda_stream))
    return [s["table"], s["free"], o["left"], o["cu"], o["kv"], o["pos"], o["slot"]]


def _own_write(s):
    ld = s["hkv"] * s["d"]
    k, v = s["kv"][:, 0], s["kv"][:, 1]
    _ok(_lib().hbk_kv_write_q4(_p(k), 2 * ld, _p(v), 2 * ld, _p(s["slots"]), _p(s["planes"][0]), _p(s["planes"][1]), _p(s["seen"][0]), ld, _p(s["seen"][1]), ld,
                               s["t"], s["hkv"], s["d"], PAGE, s["pages"], torch.cuda.current_stream().cuda_stream))
    return s["seen"]


def _own_attn(s):
    l, stream = _lib(), torch.cuda.current_stream().cuda_stream
    if s["work"] is None:
        s["work"] = torch.empty(l.hbk_attn_paged_q4_workspace_floats(s["seqs"], s["t"], s["most_rows"], s["longest"], s["hq"], s["hkv"], s["d"], s["split"], s["window"]),
                                device="cuda", dtype=torch.float32)
    _ok(l.hbk_attn_paged_q4(_p(s["q"]), s["hq"] * s["d"], _p(s["k"]), _p(s["v"]), _p(s["table"]), s["width"], _p(s["kv"]), _p(s["cu"]), _p(s["out"]), s["hq"] * s["d"],
                            _p(s["work"]), s["seqs"], s["t"], s["most_rows"], s["longest"], s["hq"], s["hkv"], s["d"], PAGE, s["split"], s["scale"], s["pages"], s["window"],
                            s["softcap"], _p(s["sink"]), stream))
    return s["out"]


def _own_product(s):
    epi = {"none": 0, "bias": 1, "resid": 3, "bias_resid": 4, "f32": 6}[s["epi"]]
    _ok(_lib().hbk_gemm_q4(_p(s["x"]), s["k"], _p(s["w"]), _p(s["out"]), s["n"], _p(s["r"]), s["n"], _p(s["bias"]), s["m"], s["n"], s["k"], epi,
                           torch.cuda.current_stream().cuda_stream))
    return s["out"]


def run(state):
    kind = state["kind"]
    if own:
        return {"tables": _own_tables, "write": _own_write, "attn": _own_attn, "product": _own_product}[kind](state)
    return {"tables": _plain_tables, "write": _plain_write, "attn": _plain_attn, "product": _plain_product}[kind](state)


# ------------------------------------------------------------------ work and values in 64 bits
def work(case):
    if case["kind"] == "tables":
        b, t = case["reqs"], case["reqs"] * case["longest_new"]
        return dict(bytes=4 * (4 * b + 1 + 2 * t + t // PAGE), flops=10 * (b + t))
    if case["kind"] == "write":
        n = case["rows"] * case["hkv"] * case["d"] * 2
        return dict(bytes=n * 2 + n * 9 // 16 + n * 2 + 4 * case["rows"], flops=6 * n)
    if case["kind"] == "attn":
        lens, rows = _portions(case)
        w, hq, hkv, d = case["window"], case["hq"], case["hkv"], case["d"]
        read = sum(min(n, w + r - 1) if w else n for n, r in zip(lens, rows))
        pairs = sum(sum(min(n - r + i + 1, w) if w else n - r + i + 1 for i in range(r)) for n, r in zip(lens, rows))
        return dict(bytes=read * hkv * (d + d // 8) + 4 * sum(rows) * hq * d, flops=4 * pairs * hq * d)
    m, n, k = case["m"], case["n"], case["k"]
    wide = 4 if case["epi"] == "f32" else 2
    return dict(bytes=n * k * 9 // 16 + 2 * m * k + m * n * (wide + (2 if "resid" in case["epi"] else 0)), flops=2 * m * n * k)


def _exact_values(plane, d, keys):
    """fp64 [..., 64, D]: each entry by the place of its nibble."""
    pos, e = torch.arange(PAGE, device="cuda")[:, None], torch.arange(d, device="cuda")[None]
    j, r = e // 32, e % 32
    if keys:
        i = r % 8
        nib = torch.where(i % 2 == 0, i // 2, 4 + i // 2)
        byte = pos * (d // 2) + (r // 8) * (d // 8) + j * 4 + nib // 2
    else:
        pair, g, nib = pos // 2, r // 4, r % 4
        place = g ^ ((pair % 4) * 2 if d == 128 else (pair // 2 % 2) * 4)
        byte = pair * d + place * (d // 8) + j * 4 + (pos % 2) * 2 + nib // 2
    code = (plane[..., byte.flatten()].long() >> (4 * (nib % 2) + 0 * byte).flatten()) % 16
    scale = plane[..., PAGE * d // 2:].contiguous().view(BF).double().unflatten(-1, (PAGE, d // 32)).repeat_interleave(32, -1)
    return (code - 8).double().unflatten(-1, (PAGE, d)) * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return None
    if case["kind"] == "write":
        x = s["kv"].double().reshape(-1, 32)
        big = x.abs().max(-1).values[:, None]
        first = torch.where(x.abs() == big, torch.arange(32, device="cuda"), 32).min(-1).values
        d = (x[torch.arange(len(x), device="cuda"), first] / -8).to(BF).double()[:, None]
        c = (x / torch.where(d == 0, 1, d) + 8.5).floor().clamp(0, 15)
        y = torch.where(d == 0, 0, d * (c - 8)).view(s["kv"].shape)
        return [y[:, 0], y[:, 1]]
    if case["kind"] == "product":
        full = []
        e = torch.arange(128, device="cuda")
        i = e % 8
        nib = torch.where(i % 2 == 0, i // 2, 4 + i // 2)
        byte = (e % 32 // 8) * 16 + e // 32 * 4 + nib // 2
        for rows in range(16):
            code = s["w"][:, :, rows * 64 + byte].long() >> (4 * (nib % 2)) & 15
            scale = s["w"][:, :, 1024 + 8 * rows:1032 + 8 * rows].contiguous().view(torch.float16).double().repeat_interleave(32, -1)
            full.append(((code - 8).double() * scale).flatten(1))
        y = s["x"].double() @ torch.stack(full, 1).flatten(0, 1)[:s["n"], :s["k"]].T
        for more in (s["bias"], s["r"]):
            if more is not None:
                y = y + more.double()
        return y
    lens, rows = _portions(case)
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        ids = s["table"][b, :-(-n // PAGE)].long()
        j, last = torch.arange(n, device="cuda"), torch.arange(n - r, n, device="cuda")[:, None, None]
        hidden = (j > last) | ((j <= last - s["window"]) if s["window"] > 0 else (j < 0))
        for h in range(s["hkv"]):
            k, v = (_exact_values(s[x][ids, h], s["d"], x == "k").flatten(0, 1)[:n] for x in ("k", "v"))
            heads = slice(h * s["hq"] // s["hkv"], (h + 1) * s["hq"] // s["hkv"])
            x = torch.einsum("ihd,jd->ihj", s["q"][at:at + r, heads].double(), k) * s["scale"]
            if s["softcap"] > 0:
                x = s["softcap"] * torch.tanh(x / s["softcap"])
            e = torch.where(hidden, 0, torch.exp(x))
            total = e.sum(-1, keepdim=True)
            if s["sink"] is not None:
                total = total + torch.exp(s["sink"][heads].double())[:, None]
            out[at:at + r, heads] = torch.einsum("ihj,jd->ihd", e, v) / total
        at += r
    return out
