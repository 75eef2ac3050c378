"""Rows coded in 8 bits, products of such rows, and scores of given tokens (from a head's product and from logits), each against plain 64-bit forms, and together."""
import ctypes
import math

import pytest
import torch

import helix_b200 as hb

pytestmark = pytest.mark.gpu
BF, DEV = torch.bfloat16, "cuda"
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def L():
    l = hb.lib()
    assert l.hbk_init() == 0, l.hbk_last_error()
    return l


def p(t):
    return t.data_ptr() if t is not None else None


def here():
    return torch.cuda.current_stream().cuda_stream


def ck(l, rc):
    assert rc == 0, (rc, l.hbk_last_error())


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(*shape, generator=gen(seed), device=DEV)


def up(n, to):
    return -(-n // to) * to


# ------------------------------------------------------------------ rows to codes
def code(L, x, seen="new", stream=None):
    """x [T, K] -> codes, scales, what they stand for; checks that nothing else is written."""
    T, K = x.shape
    ldc = up(K, 16) + 16
    codes, scales = torch.full((T + 1, ldc), 99, dtype=torch.int8, device=DEV), torch.full((T + 1,), -5.0, device=DEV)
    s = {"new": torch.full((T + 1, up(K, 8) + 8), 7.0, dtype=BF, device=DEV), "own": x, None: None}[seen]
    ck(L, L.hbk_rows_q8(p(x), int(x.dtype == torch.float32), x.stride(0), p(codes), ldc, p(scales), p(s), s.stride(0) if s is not None else 0, T, K, stream or here()))
    torch.cuda.synchronize()
    assert (codes[T] == 99).all() and (codes[:, K:] == 99).all() and scales[T] == -5
    if seen == "new":
        assert (s[T] == 7).all() and (s[:, K:] == 7).all()
    return codes[:T, :K], scales[:T], s[:T, :K] if s is not None else None


def plain_codes(x):
    """The definition in 64 bits: x / s has 48 significant bits at most that matter (24 + 8 + 24 of x, the middle and s), so its rounding decides nothing."""
    x = x.double()
    top = x.abs().max(-1).values
    s = (top.float() / torch.full((), 127.0, device=DEV)).double()  # (tensor by tensor: a quotient, rounded once)
    s = torch.where(torch.isfinite(x).all(-1), s, NAN)
    live = (s > 0)[:, None]
    c = torch.where(live, (x / s[:, None]).round().clamp(-127, 127), 0.0)
    return c.nan_to_num(0.0), s


def check_codes(x, codes, scales, seen):
    c, s = plain_codes(x)
    assert torch.equal(codes.double(), c)
    assert torch.equal(torch.nan_to_num(scales.double(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    if seen is not None:
        want = (c * s[:, None]).float().to(BF)  # (a code times a scale has 31 bits: the rounding to 24 and then to 8 that the kernel makes)
        assert torch.equal(torch.nan_to_num(seen.float(), nan=-1.0), torch.nan_to_num(want.float(), nan=-1.0))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 8), (2, 7), (3, 255), (5, 1024), (4, 1023), (33, 768), (7, 1025), (32, 4096), (3, 4095), (2, 4097), (5, 8192), (3, 8200), (2, 14336), (1, 16384), (2, 16391),
                                 (2, 40003), (1000, 136)])
def test_rows(L, T, K, f32):
    x = randn(T * 31 + K, T, up(K, 8) + 8) * torch.exp(3 * randn(K, T, 1))
    x[:, :K:17] *= 9
    x = (x if f32 else x.to(BF))[:, :K]
    check_codes(x, *code(L, x))
    check_codes(x, *code(L, x, seen=None))


def test_rows_seen_in_their_own_place(L):
    for K in (700, 5000, 33000):
        x = randn(K, 6, up(K, 8)).to(BF)[:, :K]
        was = x.clone()
        codes, scales, seen = code(L, x, seen="own")
        check_codes(was, codes, scales, seen)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("up_by", [0, 100, -60, -97, -110, -130])
def test_rows_in_the_middle_of_two_codes(L, f32, up_by):
    """The largest is 127 2^e, so s = 2^e: halves are middles, and go to the even code; their neighbours in the type go to the nearer one."""
    n = torch.arange(-126, 126, device=DEV, dtype=torch.float32) + 0.5
    x = torch.cat([torch.full((1,), 127.0, device=DEV), n, n * (1 + 2.0 ** -8), n * (1 - 2.0 ** -8), n * (1 + 2.0 ** -23), n * (1 - 2.0 ** -23)])[None].repeat(3, 1)
    x[1] *= -1
    x = (x.double() * 2.0 ** up_by).float()
    x = torch.nn.functional.pad(x if f32 else x.to(BF), (0, up(x.shape[1], 8) - x.shape[1]))
    check_codes(x, *code(L, x))


@pytest.mark.parametrize("f32", [False, True])
def test_rows_of_any_scale(L, f32):
    """Near-middles under scales of all kinds: x = (n + 1/2) s and its neighbours, s = top / 127 rounded, for many tops."""
    tops = torch.cat([torch.exp2(torch.rand(4000, generator=gen(1), device=DEV) * 250 - 126), torch.tensor([3e38, 1.2e-38, 1e-40, 1e-44, 1.4e-45], device=DEV)])
    tops = tops.to(BF).float() if not f32 else tops
    s = (tops / torch.full((), 127.0, device=DEV)).double()
    n = torch.randint(0, 127, (len(tops), 64), generator=gen(2), device=DEV) + 0.5
    x = (n * s[:, None]).float()
    bits = x.view(torch.int32)
    x = torch.cat([tops[:, None], x, (bits + 1).view(torch.float32), (bits - 1).clamp(min=0).view(torch.float32)], 1)
    x[:, 1:] = torch.minimum(x[:, 1:], tops[:, None])
    x = torch.nn.functional.pad(x, (0, up(x.shape[1], 8) - x.shape[1]))
    x = x if f32 else x.to(BF)
    check_codes(x, *code(L, x))


def test_rows_that_have_no_scale(L):
    x = randn(3, 7, 512)
    x[0] = 0
    x[1] = -0.0
    x[2, 100] = INF
    x[3, 5] = -INF
    x[4, 511] = NAN
    x[5] *= 0
    x[5, 9] = 1e-45  # the smallest there is: the quotient by 127 rounds to 0
    for y in (x, x.to(BF)):
        codes, scales, seen = code(L, y)
        check_codes(y, codes, scales, seen)
        assert (codes[:6] == 0).all() and (scales[[0, 1, 5]] == 0).all() and torch.isnan(scales[2:5]).all() and torch.isnan(seen[2:5]).all() and (codes[6] != 0).any()


@pytest.mark.parametrize("T,K", [(600, 9000), (901, 8193), (1300, 10240), (1200, 12287), (1250, 14336), (1301, 16381), (1190, 16384)])
def test_long_rows_one_after_the_other(L, T, K):
    """fp32 rows of 8193 to 16384 entries, more than the SMs take at a time: a block has several, the next on its way while it works on one."""
    x = randn(K, T, up(K, 8) + 8) * torch.exp(3 * randn(T, T, 1))
    x[T // 2, :] = 0
    x[T // 2 + 1, K - 1] = NAN
    x[T // 3, 5] = -INF
    x[T - 1, K - 1] = 1e5
    x = x[:, :K]
    check_codes(x, *code(L, x))
    check_codes(x, *code(L, x, seen=None))


def test_rows_beyond_32_bit_offsets(L):
    K, ld = 3000, 2 ** 30 + 16
    x = torch.empty(2 * ld + up(K, 8), dtype=BF, device=DEV)
    codes = torch.empty(2 * ld + up(K, 16), dtype=torch.int8, device=DEV)
    scales = torch.empty(3, device=DEV)
    rows = randn(4, 3, K).to(BF)
    for i in range(3):
        x[i * ld:i * ld + K] = rows[i]
    ck(L, L.hbk_rows_q8(p(x), 0, ld, p(codes), ld, p(scales), None, 0, 3, K, here()))
    torch.cuda.synchronize()
    got = torch.stack([codes[i * ld:i * ld + K] for i in range(3)])
    check_codes(rows, got, scales, None)


# ------------------------------------------------------------------ products
def any_codes(seed, rows, k, low=-127):
    """Codes in rows that are longer than k, full of other codes behind it."""
    c = torch.randint(low, 128, (rows, up(k, 16) + 16), generator=gen(seed), device=DEV).to(torch.int8)
    s = torch.exp(randn(seed + 1, rows)) * 1e-2
    return c, s


def product(L, x, xs, w, ws, K, epi, r=None, bias=None, out=None):
    M, N = x.shape[0], w.shape[0]
    wide = N // 2 if epi == 5 else N
    dtype = torch.float32 if epi == 6 else BF
    if out is None:
        out = torch.full((M + 1, up(wide, 8) + 8), 9.0, dtype=dtype, device=DEV)
    ck(L, L.hbk_gemm_q8(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(out), out.stride(0), p(r), r.stride(0) if r is not None else 0, p(bias), M, N, K, epi, here()))
    torch.cuda.synchronize()
    assert L.hbk_q8_status() == 0
    return out


def check_product(got, x, xs, w, ws, K, epi, r=None, bias=None):
    """Half a step is 2^-24 of the value in fp32, 2^-8 in bf16.  The whole sum is exact; its conversion and the two scales round three times, what is added once each."""
    half = 2.0 ** -24
    y = (x[:, :K].double() @ w[:, :K].double().T) * xs.double()[:, None] * ws.double()
    off = 3.01 * half * y.abs()
    if bias is not None:
        y = y + bias.double()
        off = off + half * y.abs()
    if epi == 2:
        z = y
        y = 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)
        # erfc off by 1.5e-7 and, through two approximate functions and six products, by 2^-20 of itself at most; the slope is below 1.13
        off = 1.13 * off + 0.5 * z.abs() * (1.6e-7 + 2.0 ** -20 * torch.special.erfc(z.abs() * 0.5 ** 0.5)) + 2 * half * y.abs()
    if epi == 5:
        y, off = y.unflatten(1, (-1, 2, 128)), off.unflatten(1, (-1, 2, 128))
        g, u = y.unbind(2)
        og, ou = off.unbind(2)
        # e^-g by an approximate power of two: off by 2^-21 and by the rounding of its exponent, 2^-23 |g| of itself; silu's slope is below 1.1
        a = g * torch.sigmoid(g)
        off = (1.1 * og * u.abs() + a.abs() * ou + (2.0 ** -20 + 2.0 ** -22 * g.abs()) * (a * u).abs() + 1e-37 * u.abs()).flatten(1)
        y = (a * u).flatten(1)
    if r is not None:
        y = y + r.double()
        off = off + half * y.abs()
    if epi != 6:
        off = off + 2.0 ** -8 * y.abs() + 1e-40
    bad = (got.double() - y).abs() - off
    assert (bad <= 0).all(), bad.max().item()


SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 96), (5, 130, 4096), (7, 1000, 160), (8, 64, 2048), (9, 33, 417), (13, 515, 1056), (16, 4096, 512), (17, 40, 128), (31, 100, 8961), (32, 2048, 256),
         (33, 48, 320), (64, 96, 1025), (65, 129, 31), (100, 70, 544), (128, 1000, 3000), (1, 30000, 64),  # a cluster shares K
         (129, 256, 300), (256, 50, 96), (300, 2000, 500), (1000, 100, 9000),                             # and so with more rows
         (400, 6000, 100), (400, 6003, 300), (1000, 4005, 40), (1300, 1500, 1000), (2049, 520, 272),   # tiles of one block
         (2600, 2304, 272), (2570, 2100, 1100), (5000, 4101, 130),                                        # tiles of pairs
         (154, 2722, 3033), (4194, 131, 3548), (6877, 260, 1948), (6546, 390, 1441), (6327, 392, 101), (6672, 397, 2840)]  # every shape of tile, plain and with more behind the products


@pytest.mark.parametrize("epi", [0, 1, 2, 3, 4, 6])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(L, M, N, K, epi):
    (x, xs), (w, ws) = any_codes(M, M, K), any_codes(N + 7, N, K)
    ws = ws * K ** -0.5
    bias = randn(1, up(N, 8)).to(BF)[:N] if epi in (1, 2, 4) else None
    r = randn(2, M, up(N, 8) + 16).to(BF)[:, :N] if epi in (3, 4) else None
    out = product(L, x, xs, w, ws, K, epi, r=r, bias=bias)
    check_product(out[:M, :N], x, xs, w, ws, K, epi, r, bias)
    assert (out[M] == 9).all() and (out[:, N:] == 9).all()


@pytest.mark.parametrize("M,N,K", [(1, 256, 64), (5, 512, 4096), (32, 2048, 1000), (128, 768, 70), (130, 256, 500), (300, 1024, 333), (700, 4608, 128), (2600, 2560, 272)])
def test_product_gated(L, M, N, K):
    (x, xs), (w, ws) = any_codes(M, M, K), any_codes(N + 7, N, K)
    ws = ws * K ** -0.5
    out = product(L, x, xs, w, ws, K, 5)
    check_product(out[:M, :N // 2], x, xs, w, ws, K, 5)
    assert (out[M] == 9).all() and (out[:, N // 2:] == 9).all()


@pytest.mark.parametrize("M,N", [(6, 300), (300, 2000), (400, 6000), (2600, 2304)])
def test_product_residual_in_place_and_again(L, M, N):
    K = 700
    (x, xs), (w, ws) = any_codes(M, M, K), any_codes(N + 7, N, K)
    r = randn(5, M, up(N, 8)).to(BF)
    out = r.clone()
    product(L, x, xs, w, ws, K, 3, out=out, r=out)
    check_product(out[:, :N], x, xs, w, ws, K, 3, r[:, :N])
    a, b = product(L, x, xs, w, ws, K, 6), product(L, x, xs, w, ws, K, 6)
    assert torch.equal(a, b)


@pytest.mark.parametrize("epi", [1, 2, 4, 5, 6])
def test_product_bits_do_not_depend_on_the_other_rows(L, epi):
    """A row's sums are whole numbers: alone, among few and among many it has the same bits, whichever kernel it goes through."""
    N, K = 2304, 1000
    (x, xs), (w, ws) = any_codes(3, 2600, K), any_codes(4, N, K)
    bias = randn(1, N).to(BF) if epi in (1, 2, 4) else None
    r = randn(2, 2600, N).to(BF) if epi == 4 else None
    whole = product(L, x, xs, w, ws, K, epi, r=r, bias=bias)[:2600]
    for rows in (slice(0, 1), slice(70, 100), slice(1000, 1300), slice(2000, 2500)):
        part = product(L, x[rows], xs[rows].contiguous(), w, ws, K, epi, r=r[rows] if r is not None else None, bias=bias)
        assert torch.equal(part[:-1], whole[rows])


@pytest.mark.parametrize("epi", [0, 1, 2, 3, 4, 6])
@pytest.mark.parametrize("N", [2284, 2305, 2335])
def test_product_bits_do_not_depend_on_the_other_rows_in_the_last_columns(L, N, epi):
    """Nor do they in the columns of a last group that is not whole."""
    K = 1000
    (x, xs), (w, ws) = any_codes(3, 2600, K), any_codes(4, N, K)
    bias = randn(1, up(N, 8)).to(BF)[:N] if epi in (1, 2, 4) else None
    r = randn(2, 2600, up(N, 8)).to(BF)[:, :N] if epi in (3, 4) else None
    whole = product(L, x, xs, w, ws, K, epi, r=r, bias=bias)[:2600, :N]
    for rows in (slice(0, 1), slice(70, 100), slice(1000, 1300), slice(2000, 2500)):
        part = product(L, x[rows], xs[rows].contiguous(), w, ws, K, epi, r=r[rows] if r is not None else None, bias=bias)
        assert torch.equal(part[:-1, :N], whole[rows])


@pytest.mark.parametrize("epi", [0, 1, 3, 4, 6])
def test_product_zeros_have_the_same_sign_in_every_kernel(L, epi):
    """Scales below 0, and such that products of them have no number: -0 as 0 times those is, whatever the other rows."""
    M, N, K = 2600, 2304, 100
    (x, xs), (w, ws) = any_codes(3, M, K), any_codes(4, N, K)
    x[::3] = 0
    xs[:2000], ws[::2] = -xs[:2000], -ws[::2]
    xs[1000:], ws[1::4] = xs[1000:] * 1e-22, ws[1::4] * 1e-23
    bias = torch.full((N,), -0.0, dtype=BF, device=DEV) if epi in (1, 4) else None
    r = torch.full((M, N), -0.0, dtype=BF, device=DEV) if epi in (3, 4) else None
    bits = torch.int32 if epi == 6 else torch.int16
    whole = product(L, x, xs, w, ws, K, epi, r=r, bias=bias)[:M, :N].contiguous().view(bits)
    assert (whole == torch.iinfo(bits).min).sum() > 1000  # -0
    for rows in (slice(0, 3), slice(1000, 1030), slice(1900, 2028), slice(2000, 2500)):
        part = product(L, x[rows], xs[rows].contiguous(), w, ws, K, epi, r=r[rows] if r is not None else None, bias=bias)
        assert torch.equal(part[:-1, :N].contiguous().view(bits), whole[rows])


@pytest.mark.parametrize("M", [3, 130, 2600])
@pytest.mark.parametrize("a,b", [(-128, -128), (-128, 127), (127, 127)])
def test_product_of_the_largest_sums(L, M, a, b):
    """|sums| up to 2^31 - 2^18: nothing wraps at the longest K."""
    N, K = (2304 if M == 2600 else 40), 131056
    x, w = torch.full((M, K), a, dtype=torch.int8, device=DEV), torch.full((N, K), b, dtype=torch.int8, device=DEV)
    xs, ws = torch.full((M,), 0.5, device=DEV), torch.full((N,), 2.0 ** -20, device=DEV)
    out = product(L, x, xs, w, ws, K, 6)
    want = torch.tensor(a * b * K, dtype=torch.float64).float().item() * 2.0 ** -21
    assert (out[:M, :N] == want).all()


def test_product_keeps_scales_that_are_none_in_their_rows(L):
    for M, N in ((9, 64), (300, 300), (2600, 2304)):
        K = 256
        (x, xs), (w, ws) = any_codes(9, M, K), any_codes(10, N, K)
        xs[2], xs[8] = NAN, 0.0
        ws[5] = INF
        out = product(L, x, xs, w, ws, K, 6)[:M, :N]
        assert torch.isnan(out[2]).all() and (out[8, torch.arange(N) != 5] == 0).all() and not torch.isfinite(out[:, 5]).any()
        rows = [i for i in range(M) if i not in (2, 8)]
        cols = [j for j in range(N) if j != 5]
        check_product(out[rows][:, cols], x[rows], xs[rows], w[cols], ws[cols], K, 6)


def test_product_of_many_columns(L):
    """More tiles of columns than a launch of clusters has room for, and offsets past 32 bits."""
    M, N, K = 260, 9 * 2 ** 20, 16
    (x, xs), (w, ws) = any_codes(11, M, K), any_codes(12, N, K)
    out = product(L, x, xs, w, ws, K, 0)
    for cols in (slice(0, 1000), slice(N // 2, N // 2 + 1000), slice(N - 1000, N)):
        check_product(out[:M, cols], x, xs, w[cols], ws[cols], K, 0)
    one = product(L, x[:1], xs[:1], w, ws, K, 0)
    assert torch.equal(one[0, :N], out[0, :N])


@pytest.mark.parametrize("sms", [1, 2, 3])
def test_product_within_few_sms(L, sms):
    """A caller's share of the SMs (hb::sm_limit, of its thread) may be as small as one."""
    limit = L._ZN2hb8sm_limitEv
    limit.restype = ctypes.POINTER(ctypes.c_int)
    try:
        for M, N, K in ((5, 300, 700), (100, 300, 700), (300, 515, 300)):
            (x, xs), (w, ws) = any_codes(1, M, K), any_codes(2, N, K)
            limit()[0] = sms
            out = product(L, x, xs, w, ws, K, 0)
            limit()[0] = 0
            check_product(out[:M, :N], x, xs, w, ws, K, 0)
    finally:
        limit()[0] = 0


# ------------------------------------------------------------------ scores from a head's product
def exact_scores(z, targets):
    lse = torch.logsumexp(z, -1)
    q = torch.exp(z - lse[:, None])
    entropy = -(torch.special.xlogy(q, q)).sum(-1)
    ok = (targets >= 0) & (targets < z.shape[1])
    at = z.gather(1, targets.long().clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    return torch.where(ok, at - lse, -INF), entropy


def head(L, x, xs, w, ws, targets, H, scale=1.0, cap=0.0, want=("lp", "entropy")):
    T, V = x.shape[0], w.shape[0]
    out = {k: torch.full((T + 1,), 5.0, device=DEV) if k in want else None for k in ("lp", "entropy")}
    n = L.hbk_head_scores_workspace_floats(T, V)
    work = torch.full((n + 16,), NAN, device=DEV)
    ck(L, L.hbk_head_scores(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(targets), p(out["lp"]), p(out["entropy"]), p(work), T, V, H, scale, cap, here()))
    torch.cuda.synchronize()
    assert L.hbk_q8_status() == 0 and torch.isnan(work[n:]).all()
    for v in out.values():
        assert v is None or v[T] == 5
    return [None if v is None else v[:T] for v in out.values()]


def check_head(lp, entropy, x, xs, w, ws, targets, H, scale=1.0, cap=0.0):
    """A logit of H bf16 products is off by 2^-22 of the products' mass for every 16 that are added at a time, one of codes by five roundings; a score by twice the largest of them and the
    sums' own roundings: an entropy's weights change by as much, each times its distance from the mean, log V at most on the average."""
    x, w = x[:, :H].double(), w[:, :H].double()
    T, V = x.shape[0], w.shape[0]
    if xs is None:
        z = scale * (x @ w.T)
        off = abs(scale) * (x.abs() @ w.abs().T) * (H / 16 + 4) * 2.0 ** -22
    else:
        z = scale * (x @ w.T) * xs.double()[:, None] * ws.double()
        off = 5 * 2.0 ** -24 * z.abs()
    if cap > 0:
        z = cap * torch.tanh(z / cap)
        off = off + 2.0 ** -20 * z.abs()  # (1 - 2 / (e^2y + 1) with two approximate functions is off by 2^-22, and 1/4 at least)
    worst = off.max(-1).values
    a, b = exact_scores(z, targets if targets is not None else torch.zeros(T, dtype=torch.int32, device=DEV))
    sums = 2.0 ** -18 + 2.0 ** -23 * z.abs().max(-1).values  # (up to 300 terms one after the other, each off by 2^-22 and by its exponent's rounding)
    if lp is not None:
        assert torch.equal(torch.isinf(lp), torch.isinf(a))
        bad = ((lp.double() - a).abs() - 2 * worst - sums).nan_to_num(-1.0)
        assert (bad <= 0).all(), bad.max().item()
    if entropy is not None:
        bad = (entropy.double() - b).abs() - 2 * worst * (1 + math.log(V)) - 2 * sums * (1 + math.log(V))
        assert (bad <= 0).all(), bad.max().item()


HEADS = [(1, 1, 8), (1, 2, 1), (3, 127, 64), (7, 1000, 100), (32, 5003, 256), (64, 129, 4096), (127, 300, 72), (128, 20000, 128), (129, 255, 64), (200, 30522, 768), (256, 4000, 500), (257, 1001, 264),
         (600, 5003, 1000), (1100, 257, 33),                        # blocks' tiles
         (250, 9500, 2100), (500, 20100, 2100), (700, 18900, 2100)]  # pairs'


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("T,V,H", HEADS)
def test_head(L, T, V, H, q8):
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    targets[::5] = V - 1
    if q8:
        (x, xs), (w, ws) = any_codes(T, T, H), any_codes(V + 9, V, H)
        xs, ws = xs * 3, ws * H ** -0.5
    else:
        x, w = randn(T, T, up(H, 8) + 8).to(BF), (randn(V, V, up(H, 8) + 8) * 2.5 * H ** -0.5).to(BF)
        xs = ws = None
    for scale, cap in ((1.0, 0.0), (-0.7, 0.0), (0.5, 2.0)):
        lp, entropy = head(L, x, xs, w, ws, targets, H, scale, cap)
        check_head(lp, entropy, x, xs, w, ws, targets, H, scale, cap)


def test_head_parts_that_are_not_wanted(L):
    for T in (5, 300):
        V, H = 700, 64
        x, w = randn(1, T, H).to(BF), (randn(2, V, H) * 0.3).to(BF)
        targets = torch.randint(0, V, (T,), generator=gen(3), device=DEV).int()
        lp, entropy = head(L, x, None, w, None, targets, H)
        a, none = head(L, x, None, w, None, targets, H, want=("lp",))
        assert none is None and torch.equal(a, lp)
        none, b = head(L, x, None, w, None, None, H, want=("entropy",))
        assert none is None and torch.equal(b, entropy)


def test_head_targets_that_are_none(L):
    for T in (6, 400):
        V, H = 300, 64
        x, w = randn(1, T, H).to(BF), (randn(2, V, H) * 0.3).to(BF)
        targets = torch.randint(0, V, (T,), generator=gen(3), device=DEV).int()
        targets[0], targets[1], targets[2], targets[3] = -1, V, V + 20, 2 ** 31 - 1
        lp, entropy = head(L, x, None, w, None, targets, H)
        assert (lp[:4] == -INF).all() and torch.isfinite(lp[4:]).all()
        check_head(lp, entropy, x, None, w, None, targets, H)


@pytest.mark.parametrize("T", [9, 400])
def test_head_keeps_infinities_and_nan_in_their_rows(L, T):
    V, H = 500, 64
    x, w = randn(1, T, H).to(BF), (randn(2, V, H) * 0.3).to(BF)
    targets = torch.randint(0, V, (T,), generator=gen(3), device=DEV).int()
    good = head(L, x, None, w, None, targets, H)
    y = x.clone()
    y[3, 5], y[6, 60] = NAN, INF
    bad = head(L, y, None, w, None, targets, H)
    rows = [i for i in range(T) if i not in (3, 6)]
    for a, b in zip(good, bad):
        assert torch.equal(a[rows], b[rows]) and torch.isnan(b[[3, 6]]).all()


@pytest.mark.parametrize("T", [4, 300])
@pytest.mark.parametrize("scale", [0.0, 200.0, 1e-30])
def test_head_flat_and_steep_rows(L, T, scale):
    V, H = 3000, 128
    x, w = randn(1, T, H).to(BF), (randn(2, V, H) * 0.3).to(BF)
    targets = torch.randint(0, V, (T,), generator=gen(3), device=DEV).int()
    lp, entropy = head(L, x, None, w, None, targets, H, scale=scale)
    check_head(lp, entropy, x, None, w, None, targets, H, scale=scale)
    if scale < 1:
        assert (lp + math.log(V)).abs().max() < 1e-5 and (entropy - math.log(V)).abs().max() < 1e-5


@pytest.mark.parametrize("T", [4, 100, 300])
@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-30, 0.01, 0.3, 5.0, 1e4, 1e30, 3.4e38])
def test_head_caps_of_any_size(L, T, cap):
    V, H = 3000, 128
    x, w = randn(1, T, H).to(BF), (randn(2, V, H) * 0.3).to(BF)
    x[2] = 0  # logits of 0 stay 0
    targets = torch.randint(0, V, (T,), generator=gen(3), device=DEV).int()
    cap = torch.tensor(cap, dtype=torch.float32).item()  # (as the call takes it)
    lp, entropy = head(L, x, None, w, None, targets, H, cap=cap)
    check_head(lp, entropy, x, None, w, None, targets, H, cap=cap)
    assert (lp[2] + math.log(V)).abs() < 1e-5


def test_head_again_is_the_same(L):
    for T in (30, 700):
        V, H = 9000, 512
        x, w = randn(1, T, H).to(BF), (randn(2, V, H) * 0.1).to(BF)
        targets = torch.randint(0, V, (T,), generator=gen(3), device=DEV).int()
        a, b = head(L, x, None, w, None, targets, H), head(L, x, None, w, None, targets, H)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def plain_head(w0, T, H, q8, scale=1.0):
    """A head whose logits are scale times w0 [V], whole numbers of seven bits, in every row, through the call."""
    V = len(w0)
    x, w = torch.zeros(T, up(H, 16), dtype=torch.int8, device=DEV), torch.zeros(V, up(H, 16), dtype=torch.int8, device=DEV)
    x[:, 0], w[:, 0] = 1, w0
    ones = torch.ones(max(T, V), device=DEV)
    z = scale * w0.double()[None].expand(T, V)
    return (x, ones[:T], w, ones[:V], z) if q8 else (x.to(BF), None, w.to(BF), None, z)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("w0,last", [(1, 2), (-3, -1)])
@pytest.mark.parametrize("T,V", [(9, 1001), (100, 1001), (100, 30522), (300, 1001), (300, 30522), (700, 33), (2100, 30522)])
def test_head_of_very_large_logits(L, T, V, w0, last, q8):
    """Logits 1e13 apart, the two largest the last: what is not there (columns from V on) has no weight however large the others are."""
    H = 64
    logits = torch.full((V,), w0, dtype=torch.int8, device=DEV)
    logits[-2:] = last
    x, xs, w, ws, z = plain_head(logits, T, H, q8, 1e13)
    targets = torch.full((T,), V - 1, dtype=torch.int32, device=DEV)
    targets[1::2] = 0
    lp, entropy = head(L, x, xs, w, ws, targets, H, scale=1e13)
    a, b = exact_scores(z - z.max(), targets)  # (whole numbers of 1e13: exact)
    # two weights of 1 and their logarithm: four roundings of numbers below 2; a far token's score is its distance, rounded with both logits
    assert ((lp.double() - a).abs() <= 2.0 ** -21 + 2.0 ** -21 * a.abs()).all() and (entropy.double() - b).abs().max() <= 2.0 ** -21


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("T,V", [(9, 1000), (9, 3), (64, 40001), (100, 1000), (300, 1001), (400, 3), (2100, 30522)])
def test_head_logits_that_are_minus_infinity(L, T, V, cap, q8):
    """Beside others a token whose logit is -inf has no weight (a cap makes it -cap): first, last, between others, and in a group of columns alone."""
    H = 72
    none = sorted({0, V // 2, *range(32, min(V - 1, 64)), *range(128, min(V - 1, 384)), V - 1} - {1})
    if q8:
        (x, xs), (w, ws) = any_codes(T, T, H), any_codes(V + 9, V, H)
        xs, ws = xs * 3, ws * H ** -0.5
        x[:, :H] = x[:, :H].abs().clamp(min=1)
        w[none, :H] = -w[none, :H].abs().clamp(min=1)
        ws[none] = INF
        z = (x[:, :H].double() @ w[:, :H].double().T) * xs.double()[:, None] * ws.double()
    else:
        x, w, xs, ws = randn(T, T, up(H, 8)).abs().to(BF) + 0.5, (randn(V, V, up(H, 8)) * 2.5 * H ** -0.5).to(BF), None, None
        w[none, 7] = -INF
        z = x[:, :H].double() @ w[:, :H].double().T
    assert torch.equal(torch.isinf(z), torch.isin(torch.arange(V, device=DEV), torch.tensor(none, device=DEV))[None].expand(T, V)) and (z < INF).all()
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    targets[0], targets[1], targets[2] = V // 2, V - 1, 1
    lp, entropy = head(L, x, xs, w, ws, targets, H, cap=cap)
    if cap:
        z = cap * torch.tanh(z / cap)
    a, b = exact_scores(z, targets)
    seen = ~torch.isinf(z[0])
    # (as check_head, of the logits that there are)
    if q8:
        off = (5 * 2.0 ** -24 + 2.0 ** -20) * z.abs().nan_to_num(posinf=0.0)
    else:
        off = ((x[:, :H].double().abs() @ w[:, :H].double().abs().nan_to_num(posinf=0.0).T) * (H / 16 + 4) * 2.0 ** -22 + 2.0 ** -20 * z.abs().nan_to_num(posinf=0.0))
    worst, sums = off[:, seen].max(-1).values, 2.0 ** -18 + 2.0 ** -23 * z[:, seen].abs().max(-1).values
    assert torch.equal(torch.isinf(lp), torch.isinf(a)) and not torch.isnan(lp).any()
    assert ((lp.double() - a).abs() <= 2 * worst + sums)[~torch.isinf(a)].all()
    assert ((entropy.double() - b).abs() <= 2 * (worst + sums) * (1 + math.log(V))).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("T,V", [(5, 1000), (100, 1000), (300, 1000), (300, 2001)])
def test_head_of_nothing_but_minus_infinity(L, T, V, q8):
    H = 64
    x, xs, w, ws, _ = plain_head(torch.full((V,), -1, dtype=torch.int8, device=DEV), T, H, q8)
    if q8:
        ws = torch.full((V,), INF, device=DEV)
    else:
        w[:, 0] = -INF
    lp, entropy = head(L, x, xs, w, ws, torch.zeros(T, dtype=torch.int32, device=DEV), H)
    assert (lp == -INF).all() and (entropy == 0).all()


@pytest.mark.parametrize("T", [5, 100, 300])
def test_head_logits_whose_distance_has_no_number(L, T):
    """Finite logits at both ends of fp32: the lowest have no weight."""
    V, H = 1001, 64
    x, w = torch.zeros(T, H, dtype=BF, device=DEV), torch.zeros(V, H, dtype=BF, device=DEV)
    x[:, 0] = 1
    w[:, 0] = -3e38
    w[500, 0] = w[V - 1, 0] = 3e38
    targets = torch.full((T,), 500, dtype=torch.int32, device=DEV)
    lp, entropy = head(L, x, None, w, None, targets, H)
    assert (lp + math.log(2)).abs().max() <= 2.0 ** -21 and (entropy - math.log(2)).abs().max() <= 2.0 ** -21


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("T,V,H", [(1, 151936, 72), (16, 40000, 256), (33, 58000, 100), (64, 128256, 64)])
def test_head_of_few_rows_with_many_tiles_for_each_block(L, T, V, H, q8):
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    targets[::5] = V - 1
    if q8:
        (x, xs), (w, ws) = any_codes(T, T, H), any_codes(V + 9, V, H)
        xs, ws = xs * 3, ws * H ** -0.5
    else:
        x, w = randn(T, T, up(H, 8) + 8).to(BF), (randn(V, V, up(H, 8) + 8) * 2.5 * H ** -0.5).to(BF)
        xs = ws = None
    for scale, cap in ((1.0, 0.0), (0.5, 2.0)):
        lp, entropy = head(L, x, xs, w, ws, targets, H, scale, cap)
        check_head(lp, entropy, x, xs, w, ws, targets, H, scale, cap)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("way", ["rising", "falling", "up and down", "at the end"])
@pytest.mark.parametrize("T", [1, 20, 64, 100, 300])
def test_head_of_logits_that_change_from_tile_to_tile(L, T, way, q8):
    """Logits of one tile lie far from those of the next that its block takes: sums are brought to another maximum on the way, or are not."""
    V, H = 110001, 64
    step = torch.arange(V, device=DEV) // 10000  # (148 blocks take 18944 columns at a time)
    by = {"rising": 11 * step, "falling": 110 - 11 * step, "up and down": 30 * (step // 2 % 2), "at the end": 100 * (torch.arange(V, device=DEV) >= V - 3)}[way]
    x, xs, w, ws, _ = plain_head(by.to(torch.int8), T, H, q8)
    x[:, 1:] = torch.randint(-1, 2, (T, H - 1), generator=gen(1), device=DEV).to(x.dtype)
    w[:, 1:] = (torch.rand(V, H - 1, generator=gen(2), device=DEV) < 0.06).to(w.dtype)
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    targets[0] = V - 1
    lp, entropy = head(L, x, xs, w, ws, targets, H)
    check_head(lp, entropy, x, xs, w, ws, targets, H)


@pytest.mark.parametrize("T,piece", [(48, 256), (120, 256), (512, 512)])
def test_head_of_bf16_is_as_near_as_its_pieces_make_it(L, T, piece):
    """Sixteen products at a time are added to a sum, which is cut off at its last place (2^-23 of it at most, half of that on the average) each time, until a piece of K is full; the pieces are
    added in fp32.  A score is off by its token's logit and by the weighted mean of all: 2e-5 and less.  (In one piece of 4096 older and larger sums are cut off: 2.5e-5 and more.)"""
    V, H = 3000, 4096
    x, w = randn(T, T, H).to(BF), (randn(V, V, H) * 2.5 * H ** -0.5).to(BF)
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    xd, wd = x.double(), w.double()
    z, off, bound = torch.zeros(T, V, dtype=torch.float64, device=DEV), torch.zeros(T, V, dtype=torch.float64, device=DEV), {}
    for k0 in range(0, H, piece):
        part = torch.zeros_like(z)
        for k in range(k0, k0 + piece, 16):
            part += xd[:, k:k + 16] @ wd[:, k:k + 16].T
            off += 2.0 ** -24 * part.abs()
        z += part
        off += 2.0 ** -24 * z.abs()
    lp, entropy = head(L, x, None, w, None, targets, H)
    a, b = exact_scores(z, targets)
    q = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
    tol = off.gather(1, targets.long()[:, None])[:, 0] + (q * off).sum(-1) + 2.0 ** -22 * (1 + a.abs())  # (and the sums of exponentials: 2^-22 of theirs on the average)
    err = lp.double() - a
    assert err.square().mean().sqrt() <= tol.square().mean().sqrt() and err.mean().abs() <= tol.mean(), (err.square().mean().sqrt().item(), tol.square().mean().sqrt().item())
    assert tol.square().mean().sqrt() < 3e-5
    mean = ((q * (z - (q * z).sum(-1, keepdim=True))).abs() * off).sum(-1) + 2.0 ** -21 * (1 + math.log(V))  # (an entropy's slope: a weight times its distance from the mean)
    gone = entropy.double() - b
    assert gone.square().mean().sqrt() <= mean.square().mean().sqrt(), (gone.square().mean().sqrt().item(), mean.square().mean().sqrt().item())


# ------------------------------------------------------------------ scores from logits
def scores(L, x, targets, top, V, want=("lp", "rank", "entropy", "top_lp")):
    T = x.shape[0]
    o = dict(lp=torch.full((T + 1,), 5.0, device=DEV), rank=torch.full((T + 1,), -7, dtype=torch.int32, device=DEV), entropy=torch.full((T + 1,), 5.0, device=DEV),
             top_lp=torch.full((T + 1, max(top, 1)), 5.0, device=DEV))
    o = {k: v if k in want else None for k, v in o.items()}
    ids = torch.full((T + 1, max(top, 1)), -7, dtype=torch.int32, device=DEV)
    ck(L, L.hbk_token_scores(p(x), int(x.dtype == torch.float32), x.stride(0), p(targets), T, V, top, p(o["lp"]), p(o["rank"]), p(o["entropy"]), p(ids) if top else None, p(o["top_lp"]), here()))
    torch.cuda.synchronize()
    for k, v in o.items():
        if v is not None:
            assert (v[T:] == (-7 if k == "rank" else 5)).all()
    assert (ids[T:] == -7).all()
    return o["lp"][:T], o["rank"][:T], o["entropy"][:T], ids[:T, :top], o["top_lp"][:T, :top]


def order_of(z):
    """Ids by descending logit, ascending id; a NaN last."""
    return torch.sort(torch.where(torch.isnan(z), -INF, z) + 0.0, dim=-1, descending=True, stable=True).indices


def check_scores(got, x, targets, top, V):
    """Up to V / 512 terms are added one after the other, then 9 levels; each is off by 2^-22 of itself and by its exponent's rounding, 2^-23 of its distance, which is below 100 where it
    counts.  An entropy's terms are that times the distance, log V or so on the average."""
    lp, rank, entropy, ids, top_lp = got
    z = x[:, :V].double()
    a, b = exact_scores(z, targets)
    lse = torch.logsumexp(z, -1)
    sums = (V / 512 + 120) * 2.0 ** -23
    tol = sums + 2.0 ** -23 * lse.abs() + 2.0 ** -24 * a.abs().nan_to_num(posinf=0.0)
    fine = torch.isfinite(a)
    assert torch.equal(torch.isfinite(lp), fine) and ((lp.double() - a).abs() <= tol)[fine].all() and (lp[~fine] == -INF).all()
    assert ((entropy.double() - b).abs() <= 2 * sums * (1 + math.log(V)) + 2.0 ** -23 * (1 + b)).all(), (entropy.double() - b).abs().max()
    places = order_of(z)
    t = targets.long()
    ok = (t >= 0) & (t < V)
    want = (places == t.clamp(0, V - 1)[:, None]).int().argmax(-1)
    assert torch.equal(rank.long(), torch.where(ok, want, -1))
    assert torch.equal(ids.long(), places[:, :top])
    if top:
        v = z.gather(1, places[:, :top]) - lse[:, None]
        low = torch.isinf(v)
        assert torch.equal(torch.isinf(top_lp), low) and (((top_lp.double() - v).abs() <= sums + 2.0 ** -23 * (lse.abs()[:, None] + v.abs()))[~low]).all()


def logits(seed, T, V, f32, scale=2.5):
    x = randn(seed, T, up(V, 8) + 8) * scale
    return x if f32 else x.to(BF)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,V,top", [(1, 1, 0), (1, 1, 1), (2, 7, 7), (3, 8, 3), (5, 64, 64), (9, 1000, 20), (1, 4096, 5), (2, 4097, 64), (4, 8191, 1), (40, 8192, 20), (3, 16384, 33), (1, 30522, 0), (2, 32768, 64),
                                     (1, 128256, 20), (17, 151936, 20), (80, 128256, 5), (300, 33000, 64), (500, 5001, 2)])
def test_token_scores(L, T, V, top, f32):
    x = logits(T + V, T, V, f32)
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    targets[::4] = x[::4, :V].argmax(-1).int()
    check_scores(scores(L, x, targets, top, V), x, targets, top, V)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("kind", ["equal", "two", "zeros", "rising", "falling", "steps", "last", "masked", "lowest", "first step masked", "few", "none but one"])
@pytest.mark.parametrize("T,V,top", [(3, 700, 64), (2, 9000, 20), (5, 70000, 64), (450, 12000, 7)])
def test_token_scores_of_rows_in_any_order(L, kind, f32, T, V, top):
    x = logits(V, T, V, f32)
    j = torch.arange(x.shape[1], device=DEV, dtype=torch.float32)
    low = torch.finfo(x.dtype).min
    if kind == "equal":
        x[:] = -3.0
    elif kind == "two":
        x = torch.where(x > 0, torch.tensor(1.5, dtype=x.dtype, device=DEV), torch.tensor(-1.5, dtype=x.dtype, device=DEV))
    elif kind == "zeros":
        x = (x > 0).to(x.dtype) * -0.0  # zeros of both signs tie
        x[:, ::3] = 0.0
    elif kind == "rising":
        x[:] = j / V * 20
    elif kind == "falling":
        x[:] = 5 - j / V * 20
    elif kind == "steps":
        x[:] = torch.floor(j / 97) % 13
    elif kind == "last":
        x[:, V - 1] = 30
    elif kind == "masked":
        x[torch.rand(x.shape, generator=gen(5), device=DEV) < 0.95] = -INF
        x[:, 3] = 1
    elif kind == "lowest":
        x[torch.rand(x.shape, generator=gen(5), device=DEV) < 0.95] = low
        x[:, 3] = 1
    elif kind == "first step masked":
        x[:, :V - 100] = -INF
    elif kind == "few":
        x[:] = -INF
        x[:, V // 2:V // 2 + 5] = 2
    else:
        x[:] = -INF
        x[:, V - 1] = -50
    targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
    targets[0], targets[-1] = V - 1, 3
    check_scores(scores(L, x, targets, top, V), x, targets, top, V)


@pytest.mark.parametrize("f32", [False, True])
def test_token_scores_of_rows_without_a_token(L, f32):
    for T, V in ((2, 100), (3, 20000), (460, 9000)):
        x = logits(1, T, V, f32)
        x[1] = -INF
        targets = torch.randint(0, V, (T,), generator=gen(T), device=DEV).int()
        targets[1] = 7
        lp, rank, entropy, ids, top_lp = scores(L, x, targets, 5, V)
        assert lp[1] == -INF and entropy[1] == 0 and rank[1] == 7 and ids[1].tolist() == [0, 1, 2, 3, 4] and (top_lp[1] == -INF).all()
        rows = [i for i in range(T) if i != 1]
        check_scores((lp[rows], rank[rows], entropy[rows], ids[rows], top_lp[rows]), x[rows], targets[rows], 5, V)


@pytest.mark.parametrize("f32", [False, True])
def test_token_scores_of_infinities_and_nan(L, f32):
    T, V, top = 7, 21000, 9
    x = logits(2, T, V, f32)
    x[0, 20000], x[1, 5], x[2] = NAN, INF, NAN
    x[3, 17:V:2] = NAN
    x[4, :V - 3] = NAN
    targets = torch.tensor([4, 5, 9, 17, 0, 20999, 1], dtype=torch.int32, device=DEV)
    lp, rank, entropy, ids, top_lp = scores(L, x, targets, top, V)
    assert torch.isnan(lp[:5]).all() and torch.isnan(entropy[:5]).all()
    z = x[:, :V].double()
    assert rank[0] == int((z[0] > z[0, 4]).sum()) + int((z[0, :4] == z[0, 4]).sum()) and rank[1] == 0 and rank[2] == -1 and rank[3] == -1 and rank[4] == -1
    places = order_of(z)
    for b in (0, 1, 3):
        assert torch.equal(ids[b].long(), places[b, :top])
    assert (ids[2] == -1).all() and ids[4, :3].tolist() == places[4, :3].tolist() and (ids[4, 3:] == -1).all() and torch.isnan(top_lp[4]).all()
    check_scores((lp[5:], rank[5:], entropy[5:], ids[5:], top_lp[5:]), x[5:], targets[5:], top, V)


def test_token_scores_targets_that_are_none_and_parts_that_are_not_wanted(L):
    T, V = 6, 5000
    x = logits(3, T, V, True)
    targets = torch.tensor([-1, V, 2 ** 31 - 1, 5, 0, V - 1], dtype=torch.int32, device=DEV)
    got = scores(L, x, targets, 4, V)
    check_scores(got, x, targets, 4, V)
    ids = torch.zeros(T, 4, dtype=torch.int32, device=DEV)
    ck(L, L.hbk_token_scores(p(x), 1, x.stride(0), None, T, V, 4, None, None, None, p(ids), None, here()))
    entropy, lp = torch.zeros(T, device=DEV), torch.zeros(T, device=DEV)
    ck(L, L.hbk_token_scores(p(x), 1, x.stride(0), None, T, V, 0, None, None, p(entropy), None, None, here()))
    ck(L, L.hbk_token_scores(p(x), 1, x.stride(0), p(targets), T, V, 0, p(lp), None, None, None, None, here()))
    torch.cuda.synchronize()
    assert torch.equal(ids, got[3]) and torch.equal(entropy, got[2]) and torch.equal(lp, got[0])


def test_token_scores_beyond_32_bit_offsets(L):
    V, ld = 9000, 2 ** 30 + 8
    x = torch.empty(2 * ld + up(V, 8), dtype=BF, device=DEV)
    rows = randn(4, 3, V).to(BF)
    for i in range(3):
        x[i * ld:i * ld + V] = rows[i]
    targets = torch.tensor([5, 8999, 100], dtype=torch.int32, device=DEV)
    got = scores(L, x.as_strided((3, V), (ld, 1)), targets, 6, V)
    check_scores(got, rows, targets, 6, V)


# ------------------------------------------------------------------ together, in graphs, on streams
def test_scoring_a_coded_model_captured_and_replayed(L):
    """What scoring runs: hidden rows coded, a projection with a residual, its rows coded, the head's logits from the codes and their scores; the scores straight from the head beside them.
    One graph, replayed over new inputs on a stream of its own."""
    T, H, V, top = 70, 512, 4500, 8
    x, r = torch.zeros(T, H, dtype=BF, device=DEV), torch.zeros(T, H, dtype=BF, device=DEV)
    w1, wh = (randn(1, H, H) * H ** -0.5).to(BF), randn(2, V, H) * 2.5 * H ** -0.5
    c1, s1, _ = code(L, w1, seen=None)
    ch, sh, _ = code(L, wh, seen=None)
    targets = torch.zeros(T, dtype=torch.int32, device=DEV)
    c = [torch.zeros(T, H, dtype=torch.int8, device=DEV) for _ in range(2)]
    s = [torch.zeros(T, device=DEV) for _ in range(2)]
    y, z = torch.zeros(T, H, dtype=BF, device=DEV), torch.zeros(T, up(V, 8), device=DEV)
    lp, entropy, lp2, entropy2 = (torch.zeros(T, device=DEV) for _ in range(4))
    rank, ids, top_lp = torch.zeros(T, dtype=torch.int32, device=DEV), torch.zeros(T, top, dtype=torch.int32, device=DEV), torch.zeros(T, top, device=DEV)
    work = torch.empty(L.hbk_head_scores_workspace_floats(T, V), device=DEV)

    def step(st):
        ck(L, L.hbk_rows_q8(p(x), 0, H, p(c[0]), H, p(s[0]), None, 0, T, H, st))
        ck(L, L.hbk_gemm_q8(p(c[0]), H, p(s[0]), p(c1), c1.stride(0), p(s1), p(y), H, p(r), H, None, T, H, H, 3, st))
        ck(L, L.hbk_rows_q8(p(y), 0, H, p(c[1]), H, p(s[1]), None, 0, T, H, st))
        ck(L, L.hbk_gemm_q8(p(c[1]), H, p(s[1]), p(ch), ch.stride(0), p(sh), p(z), z.stride(0), None, 0, None, T, V, H, 6, st))
        ck(L, L.hbk_token_scores(p(z), 1, z.stride(0), p(targets), T, V, top, p(lp), p(rank), p(entropy), p(ids), p(top_lp), st))
        ck(L, L.hbk_head_scores(p(c[1]), H, p(s[1]), p(ch), ch.stride(0), p(sh), p(targets), p(lp2), p(entropy2), p(work), T, V, H, 1.0, 0.0, st))

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step(here())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(here())
    for i in range(4):
        x.copy_(randn(10 + i, T, H).to(BF))
        r.copy_(randn(20 + i, T, H).to(BF))
        targets.copy_(torch.randint(0, V, (T,), generator=gen(30 + i), device=DEV).int())
        graph.replay()
        torch.cuda.synchronize()
        assert L.hbk_q8_status() == 0
        check_codes(x, c[0], s[0], None)
        check_product(y, c[0], s[0], c1, s1, H, 3, r)
        check_codes(y, c[1], s[1], None)
        check_product(z[:, :V], c[1], s[1], ch, sh, H, 6)
        check_scores((lp, rank, entropy, ids, top_lp), z, targets, top, V)
        check_head(lp2, entropy2, c[1], s[1], ch, sh, targets, H)
        assert (lp - lp2).abs().max() < 1e-4 and (entropy - entropy2).abs().max() < 1e-4


def test_calls_on_two_streams_at_once(L):
    K = 1000
    cases = []
    for i, (M, N) in enumerate(((20, 3000), (2600, 2304), (300, 700), (500, 6000))):
        (x, xs), (w, ws) = any_codes(40 + i, M, K), any_codes(50 + i, N, K)
        t = torch.randint(0, N, (M,), generator=gen(i), device=DEV).int()
        cases.append((x, xs, w, ws, t, torch.zeros(M, up(N, 8), device=DEV), torch.zeros(M, device=DEV), torch.zeros(M, device=DEV), torch.empty(L.hbk_head_scores_workspace_floats(M, N), device=DEV)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for st, (x, xs, w, ws, t, out, lp, en, work) in zip(streams, cases):
            M, N = x.shape[0], w.shape[0]
            ck(L, L.hbk_gemm_q8(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(out), out.stride(0), None, 0, None, M, N, K, 6, st.cuda_stream))
            ck(L, L.hbk_head_scores(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(t), p(lp), p(en), p(work), M, N, K, 0.05, 0.0, st.cuda_stream))
    torch.cuda.synchronize()
    assert L.hbk_q8_status() == 0
    for x, xs, w, ws, t, out, lp, en, work in cases:
        check_product(out[:, :w.shape[0]], x, xs, w, ws, K, 6)
        check_head(lp, en, x, xs, w, ws, t, K, 0.05)


@pytest.mark.parametrize("M,N,K", [(5, 300, 512), (300, 1000, 512), (400, 6000, 512), (2600, 2304, 512), (250, 9500, 2100), (6877, 260, 1948), (6672, 397, 2840)])
def test_waits_that_run_out_end_the_call_and_are_said(L, M, N, K):
    """With a limit below 0 every wait is given up at once."""
    (x, xs), (w, ws) = any_codes(1, M, K), any_codes(2, N, K)
    t = torch.zeros(M, dtype=torch.int32, device=DEV)
    lp, en, work = torch.zeros(M, device=DEV), torch.zeros(M, device=DEV), torch.empty(L.hbk_head_scores_workspace_floats(M, N), device=DEV)
    out = torch.zeros(M, up(N, 8), device=DEV)
    former = L.hbk_q8_wait_cycles(-1)
    try:
        ck(L, L.hbk_gemm_q8(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(out), out.stride(0), None, 0, None, M, N, K, 6, here()))
        torch.cuda.synchronize()
        assert L.hbk_q8_status() == 702 and L.hbk_q8_status() == 0
        assert torch.isnan(out[:, :N]).all() and (out[:, N:] == 0).all()
        ck(L, L.hbk_head_scores(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(t), p(lp), p(en), p(work), M, N, K, 1.0, 0.0, here()))
        torch.cuda.synchronize()
        assert L.hbk_q8_status() == 702 and torch.isnan(lp).all() and torch.isnan(en).all()
    finally:
        L.hbk_q8_wait_cycles(former)
    ck(L, L.hbk_gemm_q8(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(out), out.stride(0), None, 0, None, M, N, K, 6, here()))
    torch.cuda.synchronize()
    assert L.hbk_q8_status() == 0
    check_product(out[:, :N], x, xs, w, ws, K, 6)


@pytest.mark.parametrize("M,N,K", [(5, 300, 20000), (60, 40000, 2048), (100, 5000, 2048), (128, 768, 9000), (300, 1000, 512), (400, 6000, 512), (2600, 2304, 512), (250, 9500, 9000), (6877, 260, 1948),
                                   (6672, 397, 2840)])
def test_waits_that_run_out_half_way_end_the_call_and_are_said(L, M, N, K):
    """With short limits waits are given up while copies and products are on their way: the call ends, what it says it lost is NaN, the rest is as it is without a limit."""
    (x, xs), (w, ws) = any_codes(1, M, K), any_codes(2, N, K)
    xb, wb = x[:, :up(K, 16)].to(BF), w[:, :up(K, 16)].to(BF)
    t = torch.randint(0, N, (M,), generator=gen(3), device=DEV).int()
    work = torch.empty(L.hbk_head_scores_workspace_floats(M, N), device=DEV)
    out, lp, en = torch.zeros(M, up(N, 8), device=DEV), torch.zeros(M, device=DEV), torch.zeros(M, device=DEV)

    said = 0

    def calls():
        yield lambda: L.hbk_gemm_q8(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(out), out.stride(0), None, 0, None, M, N, K, 6, here()), [out]
        yield lambda: L.hbk_head_scores(p(x), x.stride(0), p(xs), p(w), w.stride(0), p(ws), p(t), p(lp), p(en), p(work), M, N, K, 1e-3, 0.0, here()), [lp, en]
        yield lambda: L.hbk_head_scores(p(xb), xb.stride(0), None, p(wb), wb.stride(0), None, p(t), p(lp), p(en), p(work), M, N, K, 1e-6, 0.0, here()), [lp, en]

    for call, outs in calls():
        ck(L, call())
        torch.cuda.synchronize()
        good = [o.clone() for o in outs]
        assert L.hbk_q8_status() == 0 and all(torch.isfinite(o).all() for o in good)
        for limit in (1, 200, 700, 1500, 3000, 6000, 12000, 25000):
            former = L.hbk_q8_wait_cycles(limit)
            try:
                ck(L, call())
                torch.cuda.synchronize()
            finally:
                L.hbk_q8_wait_cycles(former)
            status = L.hbk_q8_status()
            assert status in (0, 702)
            said += status == 702
            lost = [torch.isnan(o) for o in outs]
            assert any(n.any() for n in lost) == (status == 702)
            for o, n, g in zip(outs, lost, good):
                assert torch.equal(o[~n], g[~n])
        ck(L, call())
        torch.cuda.synchronize()
        assert L.hbk_q8_status() == 0 and all(torch.equal(o, g) for o, g in zip(outs, good))
    assert said or K < 9000  # (a wait for the products of long rows takes longer than one look at it)
