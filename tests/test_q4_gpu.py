"""A step whose cache and weights are held in 4 bits, kernel by kernel and together, against plain 64-bit forms (tests/q4_ref.py)."""
import ctypes
import random

import pytest
import torch

import helix_b200 as hb
import q4_ref as ref

pytestmark = pytest.mark.gpu
BF, DEV = torch.bfloat16, "cuda"
PAGE = 64


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


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ page tables
def run_tables(L, ctx, new, table, free, num_pages, T, alias=False):
    B = len(ctx)
    c, n, tb = ints(ctx), ints(new), ints(table)
    fr = ints(list(free) + [-7] * (num_pages - len(free)))
    count = ints([len(free)])
    left = count if alias else ints([-5])
    kv = c if alias else ints([-5] * B)
    cu, pos, slot = ints([-5] * (B + 1)), ints([-5] * (T + 3)), ints([-5] * (T + 3))
    ck(L, L.hbk_page_tables(p(c), p(n), B, p(tb), tb.shape[1], p(fr), p(count), p(left), num_pages, p(cu), p(kv), p(pos), p(slot), T, PAGE, here()))
    torch.cuda.synchronize()
    table, stack, w_cu, w_kv, w_pos, w_slot = ref.page_tables(ctx, new, table, free, num_pages, T)
    assert cu.tolist() == w_cu and kv.tolist() == w_kv
    assert pos.tolist() == w_pos + [-5] * 3 and slot.tolist() == w_slot + [-5] * 3
    assert tb.tolist() == table
    assert left.item() == len(stack) and fr.tolist()[:len(stack)] == stack
    if not alias:
        assert count.item() == len(free)


def scene(rng, B, longest, longest_new, width, ended, spare):
    ctx = [rng.choice([0, 1, 63, 64, 65, rng.randint(0, longest)]) for _ in range(B)]
    new = [-1 if rng.random() < ended else rng.choice([0, 1, 1, rng.randint(0, longest_new)]) for _ in range(B)]
    held = [min(-(-c // PAGE), width) for c in ctx]
    n = sum(held) + spare + 1
    ids = rng.sample(range(n), n)
    table = []
    for h in held:
        table.append(ids[:h] + [-1] * (width - h))
        ids = ids[h:]
    return ctx, new, table, ids[:spare], n


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("B,longest_new,width,ended,spare", [
    (1, 1, 5, 0.0, 3), (1, 700, 40, 0.0, 20), (3, 64, 12, 0.3, 10), (48, 1, 12, 0.1, 48), (33, 300, 20, 0.2, 400),
    (700, 2, 12, 0.1, 300), (1023, 40, 14, 0.0, 1200), (2048, 3, 11, 0.2, 3000), (2048, 9, 11, 1.0, 0)])
def test_page_tables(L, B, longest_new, width, ended, spare, alias):
    rng = random.Random(B * 7 + longest_new)
    for k in range(3):
        ctx, new, table, free, n = scene(rng, B, 600, longest_new, width, ended, spare)
        rows = sum(max(x, 0) for x in new)
        run_tables(L, ctx, new, table, free, n, rows + [0, 5, 3000][k], alias)


@pytest.mark.parametrize("B,spare,width,cut", [(5, 0, 8, 0), (40, 7, 12, 0), (300, 60, 10, 0), (40, 100, 4, 0), (200, 900, 12, 40), (900, 11, 5, 2000), (7, 3, 6, 10 ** 6)])
def test_page_tables_refuse_what_does_not_fit(L, B, spare, width, cut):
    """Too few pages, rows of the table too short, more rows than T: those requests keep their length and have no slots; the others are served."""
    rng = random.Random(B + spare)
    for _ in range(4):
        ctx, new, table, free, n = scene(rng, B, 600, 90, width, 0.1, spare)
        run_tables(L, ctx, new, table, free, n, max(0, sum(max(x, 0) for x in new) - cut))


def test_page_tables_hold_lengths_and_page_numbers_that_are_none(L):
    run_tables(L, [-3, 70, 2 ** 31 - 1, 10], [5, 1, 1, 2 ** 31 - 1], [[-1] * 4, [9, 99, -1, -1], [-1] * 4, [2, -1, -1, -1]], [4, 5], 10, 40)


def test_page_tables_steps_replayed(L):
    """A captured step, its outputs its own next inputs: tokens are added until the pool is empty."""
    B, width, n, T = 6, 9, 40, 6
    ctx, new = ints([0, 10, 64, 127, 200, 63]), ints([1, 1, 1, 1, 0, 1])
    held = [-(-c // PAGE) for c in ctx.tolist()]
    ids = list(range(n))[::-1]
    table = [[ids.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    tb, fr, count = ints(table), ints(ids + [-1] * (n - len(ids))), ints([len(ids)])
    cu, pos, slot = ints([0] * (B + 1)), ints([0] * T), ints([0] * T)

    def call():
        ck(L, L.hbk_page_tables(p(ctx), p(new), B, p(tb), width, p(fr), p(count), p(count), n, p(cu), p(ctx), p(pos), p(slot), T, PAGE, here()))

    host = (ctx.tolist(), table, list(ids))
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call()
    for _ in range(500):
        graph.replay()
        torch.cuda.synchronize()
        t2, st2, w_cu, w_kv, w_pos, w_slot = ref.page_tables(host[0], new.tolist(), host[1], host[2], n, T)
        assert ctx.tolist() == w_kv and slot.tolist() == w_slot and tb.tolist() == t2 and count.item() == len(st2)
        host = (w_kv, t2, st2)
    assert w_slot.count(-1) > 0


# ------------------------------------------------------------------ rows into the cache
def write(L, k, v, slots, hkv, d, pages, seen="new", planes=None):
    T = slots.numel()
    planes = planes or [torch.full((pages, hkv, PAGE * d // 2 + PAGE * d // 16), 0xAB, dtype=torch.uint8, device=DEV) for _ in range(2)]
    assert L.hbk_kv_q4_plane_bytes(pages, hkv, d) == planes[0].numel()
    ks, vs = {"new": [torch.full((T, hkv * d + 8), 7.0, dtype=BF, device=DEV) for _ in range(2)], "own": [k, v], None: [None, None]}[seen]
    ck(L, L.hbk_kv_write_q4(p(k), k.stride(0), p(v), v.stride(0), p(slots), p(planes[0]), p(planes[1]), p(ks), ks.stride(0) if seen else 0, p(vs),
                            vs.stride(0) if seen else 0, T, hkv, d, PAGE, pages, here()))
    torch.cuda.synchronize()
    return planes, ks, vs


def check_written(x, seen, plane, slots, hkv, d, keys):
    T, rows = slots.numel(), x[:, :hkv * d].reshape(slots.numel(), hkv, d // 32, 32)
    c, s = ref.encode(rows)
    want = ((c - 8).double() * s[..., None]).flatten(-2)
    if seen is not None:
        assert torch.equal(torch.nan_to_num(seen[:, :hkv * d].view(T, hkv, d).float(), nan=1e38), torch.nan_to_num(want.to(BF).float(), nan=1e38))
    got_c, got_s = ref.plane_codes(plane, d, keys)
    ok = (slots >= 0) & (slots < plane.shape[0] * PAGE)
    pg, off = slots[ok].long() // PAGE, slots[ok].long() % PAGE
    finite = torch.isfinite(s[ok])
    assert torch.equal(torch.nan_to_num(got_s[pg, :, off], nan=1e38), torch.nan_to_num(s[ok], nan=1e38))
    assert torch.equal(torch.where(finite[..., None], got_c[pg, :, off].unflatten(-1, (-1, 32)), 8), c[ok])
    # what no row was written to is as it was
    left = torch.ones(plane.shape[0], PAGE, dtype=torch.bool, device=DEV)
    left[pg, off] = False
    other_c, other_s = got_c.movedim(1, 2)[left], got_s.movedim(1, 2)[left]
    fill_c, fill_s = ref.plane_codes(torch.full_like(plane[:1], 0xAB), d, keys)
    assert (other_c == fill_c.movedim(1, 2)[0, 0]).all() and (other_s == fill_s[0, 0, 0, 0]).all()


@pytest.mark.parametrize("seen", ["new", "own", None])
@pytest.mark.parametrize("T,hkv,d", [(1, 1, 64), (1, 8, 128), (3, 2, 64), (31, 3, 128), (32, 8, 128), (77, 1, 128), (130, 5, 64), (1000, 2, 128)])
def test_kv_write(L, T, hkv, d, seen):
    pages = max(4, -(-T // PAGE) + 2)
    x = torch.randn(T, 2 * hkv * d + 24, generator=gen(T + d), device=DEV).to(BF)
    k, v = x[:, 8:], x[:, 8 + hkv * d + 8:]
    slots = torch.randperm(pages * PAGE, generator=gen(5), device=DEV)[:T].int()
    if T > 2:
        slots[1], slots[T // 2] = -1, pages * PAGE
    k0, v0 = k.clone(), v.clone()
    planes, ks, vs = write(L, k, v, slots, hkv, d, pages, seen)
    check_written(k0, ks, planes[0], slots, hkv, d, True)
    check_written(v0, vs, planes[1], slots, hkv, d, False)
    if seen == "new":
        assert (ks[:, hkv * d:] == 7).all() and (vs[:, hkv * d:] == 7).all()
    if seen != "own":
        assert torch.equal(k, k0) and torch.equal(v, v0)


@pytest.mark.parametrize("T,hkv,d,start", [(1, 1, 128, 63), (2, 3, 64, 0), (130, 2, 128, 0), (131, 2, 128, 5), (64, 1, 64, 127), (77, 4, 64, 64)])
def test_kv_write_of_positions_in_a_row(L, T, hkv, d, start):
    """Prompts: neighbours share the words of values; first slots of either parity, a gap in the middle."""
    pages = (start + T) // PAGE + 2
    x = torch.randn(T, 2 * hkv * d, generator=gen(T + start), device=DEV).to(BF)
    slots = torch.arange(start, start + T, device=DEV).int()
    if T > 100:
        slots[70:] += 1
        slots[99] = -1
    planes, ks, vs = write(L, x[:, :hkv * d], x[:, hkv * d:], slots, hkv, d, pages)
    check_written(x[:, :hkv * d], ks, planes[0], slots, hkv, d, True)
    check_written(x[:, hkv * d:], vs, planes[1], slots, hkv, d, False)


@pytest.mark.parametrize("d", [64, 128])
def test_kv_write_at_the_borders_of_codes(L, d):
    """Half steps, equal magnitudes of both signs, zeros, the smallest and largest numbers, infinities and NaN, every multiple of a half scale."""
    hkv = 2
    halves = torch.arange(-16, 17, device=DEV).float() / 2
    rows = []
    for m in (-8.0, 8.0, -8.5, 7.75, -8 * 1.0078125, 12.0, 8 * 1.3359375, -3 * 2.0 ** -100, 5 * 2.0 ** 90):
        dd = float(torch.tensor(m / -8).to(BF))
        r = (halves[torch.arange(32, device=DEV) % 33] * dd)
        r[5] = m
        rows.append(r)
    rows.append(torch.zeros(32, device=DEV))
    eq = torch.ones(32, device=DEV) * 3
    eq[::2] = -3
    rows += [eq, -eq, torch.full((32,), 2.0 ** -133, device=DEV), torch.linspace(-1, 1, 32, device=DEV) * 1e-38, torch.linspace(-1, 1, 32, device=DEV) * 3e38,
             torch.linspace(-1, 1, 32, device=DEV) * 9e-40]
    for bad in (float("nan"), float("inf"), float("-inf")):
        r = torch.linspace(-1, 1, 32, device=DEV)
        r[31] = bad
        rows.append(r)
    while len(rows) * 32 % (hkv * d):
        rows.append(rows[len(rows) % 7])
    x = torch.stack(rows).view(-1, hkv * d).to(BF)
    T = x.shape[0]
    slots = ints([(7 * i) % 128 for i in range(T)])
    planes, ks, vs = write(L, x, x.flip(1).contiguous(), slots, hkv, d, 2)
    check_written(x, ks, planes[0], slots, hkv, d, True)
    check_written(x.flip(1).contiguous(), vs, planes[1], slots, hkv, d, False)


def test_kv_write_all_quotients(L):
    """Every pair of significands of entry and largest entry: a code is never on the wrong side of a half step."""
    big = (1 + torch.arange(128, device=DEV) / 128).view(128, 1, 1)
    small = (torch.arange(1, 256, device=DEV).float() / 128).view(1, 255, 1) * torch.tensor([1.0, 0.5, 0.25, 0.125], device=DEV)
    small = small.flatten(1)
    small = torch.cat([small, -small], 1)
    n = -(-small.shape[1] // 31) * 31
    small = torch.nn.functional.pad(small, (0, n - small.shape[1])).view(1, -1, 31).expand(128, -1, 31)
    small = torch.where(small.abs() > big, 0.0, small)
    x = torch.cat([small, big.expand(128, small.shape[1], 1)], -1).flatten(0, 1)
    x = torch.cat([x, -x])
    x = x[: len(x) // 4 * 4].reshape(-1, 128).to(BF)
    T = x.shape[0]
    pages = -(-T // PAGE)
    slots = torch.arange(T, device=DEV).int()
    planes, ks, vs = write(L, x, x, slots, 1, 128, pages)
    check_written(x, ks, planes[0], slots, 1, 128, True)
    check_written(x, vs, planes[1], slots, 1, 128, False)


# ------------------------------------------------------------------ attention
def attn(L, q, kp, vp, table, kv, rows, scale, window=0, softcap=0.0, sink=None, split=0, pages=None, longest=None, most=None, ldo=None, out=None, cu=True, longest_kv=None):
    T, hq, d = q.shape
    hkv = kp.shape[1]
    starts = [sum(rows[:b]) for b in range(len(rows) + 1)]
    most = most or max(max(rows), 1)
    longest_kv = longest_kv if longest_kv is not None else max(kv)
    ldo = ldo or hq * d
    out = torch.full((T, ldo), 9.0, dtype=BF, device=DEV) if out is None else out
    n = L.hbk_attn_paged_q4_workspace_floats(len(kv), T, most, longest_kv, hq, hkv, d, split, window)
    work = torch.full((n + 4,), float("nan"), device=DEV)
    cu_t, kv_t = ints(starts), ints(kv)
    ck(L, L.hbk_attn_paged_q4(p(q), q.stride(0), p(kp), p(vp), p(table), table.shape[1], p(kv_t), p(cu_t) if cu else None, p(out), ldo, p(work) if n else None,
                              len(kv), T, most, longest_kv, hq, hkv, d, PAGE, split, scale, pages or kp.shape[0], window, softcap, p(sink), here()))
    torch.cuda.synchronize()
    assert torch.isnan(work[n:]).all()
    return out


def cache(seed, lens, hkv, d, spread=1.0, spare=2, width=0):
    """Planes whose unwritten places hold NaN scales, and a shuffled table."""
    need = [-(-n // PAGE) for n in lens]
    pages = sum(need) + spare
    planes = []
    for i in range(2):
        x = torch.randn(pages, hkv, PAGE, d, generator=gen(seed + i), device=DEV)
        x *= torch.exp(spread * torch.randn(pages, hkv, PAGE, 1, generator=gen(seed + 7 + i), device=DEV)) if i else 1.0
        planes.append(ref.make_plane(x.to(BF), i == 0))
    ids = torch.randperm(pages, generator=gen(seed + 3), device=DEV).int()
    table = torch.full((len(lens), max(max(need), 1, width)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, (n, m) in enumerate(zip(lens, need)):
        table[b, :m] = ids[at:at + m]
        if n % PAGE:
            for plane in planes:
                s = plane[int(ids[at + m - 1]), :, PAGE * d // 2:].view(hkv, PAGE, -1)
                s[:, n % PAGE:] = 0xFF
        at += m
    for plane in planes:  # pages of nobody
        plane[ids[at:].long()] = 0xFF
    return planes[0], planes[1], table


def check_attn(out, want, mass, hq, d):
    """bf16 rounding of the result (2^-8 of it); every weight is rounded to fp16 by itself and again times its value scale, each by 2^-11 of it at most, so
    (1 + 2^-11)^2 - 1 < 2^-10 + 2^-21 of the sum of p |v|, or by half a step of fp16's smallest numbers, 2^-25 where the largest weight is 2^10: 2^-35 |v|, which
    2^-10 of the 2^-24 |v| in `mass` covers twice; 2^-12 of that sum for all that is done in fp32."""
    got = out[:, :hq * d].view(-1, hq, d).double()
    off = (got - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** -12) * mass + 1e-30)
    assert not torch.isnan(got).any() and (off <= 0).all(), (off.max().item(), (got - want).norm().item() / want.norm().item())


HEADS = [(1, 1), (4, 4), (4, 2), (9, 3), (8, 2), (12, 2), (16, 2), (20, 1), (32, 8)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_attention_of_single_tokens(L, hq, hkv, d):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 0, 300, 1000]
    kp, vp, table = cache(hq + d, lens, hkv, d)
    q = torch.randn(len(lens), hq, d, generator=gen(1), device=DEV).to(BF)
    for split in (0, 1, 4, 100):
        for cu in (True, False):
            out = attn(L, q, kp, vp, table, lens, [1] * len(lens), d ** -0.5, split=split, cu=cu)
            want, mass = ref.attention(q, kp, vp, table, lens, [1] * len(lens), d ** -0.5)
            check_attn(out, want, mass, hq, d)
            assert (out[10] == 0).all()


@pytest.mark.parametrize("window,softcap,sink", [(1, 0.0, False), (64, 0.0, True), (65, 30.0, False), (0, 5.0, True), (200, 50.0, True), (100000, 0.0, False)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (24, 2, 64)])
def test_attention_with_window_cap_and_sinks(L, hq, hkv, d, window, softcap, sink):
    lens = [1, 64, 130, 0, 700, 257, 64]
    rows = [1, 3, 40, 0, 17, 1, 64]
    kp, vp, table = cache(d + window, lens, hkv, d)
    q = (2 * torch.randn(sum(rows), hq, d, generator=gen(2), device=DEV)).to(BF)
    sk = torch.randn(hq, generator=gen(3), device=DEV).to(BF) * 3 if sink else None
    want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5, window, softcap, sk)
    for split in (0, 1, 3):
        out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, window, softcap, sk, split=split)
        check_attn(out, want, mass, hq, d)


@pytest.mark.parametrize("hq,hkv,d,rows", [(1, 1, 64, 9), (3, 1, 128, 50), (8, 8, 64, 33), (12, 2, 128, 70), (32, 8, 64, 129), (5, 1, 128, 300)])
def test_attention_of_portions(L, hq, hkv, d, rows):
    """Whole prompts (every position a row), a portion behind a cached prefix, a single token and nothing beside them; rows behind the last stay."""
    lens, n = [rows, 500 + rows, 77, 0, 3 * rows], [rows, rows, 1, 0, 2]
    kp, vp, table = cache(rows, lens, hkv, d)
    q = torch.randn(sum(n) + 5, hq, d, generator=gen(4), device=DEV).to(BF)
    out = attn(L, q, kp, vp, table, lens, n, d ** -0.5, ldo=hq * d + 8)
    want, mass = ref.attention(q, kp, vp, table, lens, n, d ** -0.5)
    check_attn(out[:-5], want[:-5], mass[:-5], hq, d)
    assert (out[-5:] == 9).all() and (out[:, hq * d:] == 9).all()


def test_attention_rows_before_the_first_position_are_empty(L):
    """More rows than positions: the first of them see nothing."""
    hq, hkv, d = 4, 2, 128
    kp, vp, table = cache(11, [3, 70], hkv, d)
    q = torch.randn(10, hq, d, generator=gen(4), device=DEV).to(BF)
    out = attn(L, q, kp, vp, table, [3, 70], [8, 2], d ** -0.5)
    assert (out[:5] == 0).all()
    want, mass = ref.attention(torch.cat([q[5:8], q[8:]]), kp, vp, table, [3, 70], [3, 2], d ** -0.5)
    check_attn(out[5:], want, mass, hq, d)


@pytest.mark.parametrize("hq,hkv,d,lens", [(32, 8, 128, [20000, 3, 9000]), (8, 1, 64, [70001]), (6, 2, 128, [131072, 64])])
def test_attention_over_long_caches(L, hq, hkv, d, lens):
    kp, vp, table = cache(17, lens, hkv, d, spread=0.3, width=max(lens) // PAGE + 9)
    q = (1.5 * torch.randn(len(lens), hq, d, generator=gen(5), device=DEV)).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, [1] * len(lens), d ** -0.5)
    for split in (0, 7, 64):
        check_attn(attn(L, q, kp, vp, table, lens, [1] * len(lens), d ** -0.5, split=split), want, mass, hq, d)


def test_attention_bits_depend_on_the_sequence_and_the_split_alone(L):
    hq, hkv, d = 12, 4, 128
    lens = [1500, 40, 777, 3000, 0]
    kp, vp, table = cache(23, lens, hkv, d)
    q = torch.randn(len(lens), hq, d, generator=gen(6), device=DEV).to(BF)
    full = attn(L, q, kp, vp, table, lens, [1] * 5, d ** -0.5, split=8, longest_kv=50000)
    for b in range(5):
        assert torch.equal(full[b], attn(L, q[b:b + 1], kp, vp, table[b:b + 1].clone(), lens[b:b + 1], [1], d ** -0.5, split=8)[0])
    again = attn(L, q, kp, vp, table, lens, [1] * 5, d ** -0.5, split=8, longest_kv=50000)
    assert torch.equal(full, again)


@pytest.mark.parametrize("scale", [-0.125, 0.0, 3e-30, 2.0])
def test_attention_scales(L, scale):
    """Negative, none at all (every visible position alike), next to none, large."""
    hq, hkv, d, lens, rows = 6, 2, 64, [200, 65, 1], [3, 1, 1]
    kp, vp, table = cache(3, lens, hkv, d)
    q = torch.randn(5, hq, d, generator=gen(21), device=DEV).to(BF)
    sk = torch.randn(hq, generator=gen(22), device=DEV).to(BF)
    for window, cap in ((0, 0.0), (2 ** 31 - 1, 0.0), (70, 20.0)):
        want, mass = ref.attention(q, kp, vp, table, lens, rows, scale, window, cap, sk)
        for split in (0, 1):
            check_attn(attn(L, q, kp, vp, table, lens, rows, scale, window, cap, sk, split=split), want, mass, hq, d)


def test_attention_of_many_sequences(L):
    hq, hkv, d, B = 40, 1, 64, 1500
    rng = random.Random(4)
    lens = [rng.choice([0, 1, 5, 64, 100]) for _ in range(B)]
    kp, vp, table = cache(5, lens, hkv, d)
    q = torch.randn(B, hq, d, generator=gen(23), device=DEV).to(BF)
    out = attn(L, q, kp, vp, table, lens, [1] * B, d ** -0.5)
    want, mass = ref.attention(q, kp, vp, table, lens, [1] * B, d ** -0.5)
    check_attn(out, want, mass, hq, d)


def test_planes_beyond_32_bit_offsets(L):
    """Planes of 4.8 GB: a row is written to the last page and read back by attention."""
    hkv, d, pages = 8, 128, 130000
    size = L.hbk_kv_q4_plane_bytes(pages, hkv, d)
    assert size > 2 ** 32
    planes = [torch.empty(pages, hkv, size // pages // hkv, dtype=torch.uint8, device=DEV) for _ in range(2)]
    x = torch.randn(3, 2 * hkv * d, generator=gen(24), device=DEV).to(BF)
    slots = ints([(pages - 1) * PAGE, (pages - 1) * PAGE + 1, (pages - 2) * PAGE + 63])
    ck(L, L.hbk_kv_write_q4(p(x), 2 * hkv * d, p(x[:, hkv * d:]), 2 * hkv * d, p(slots), p(planes[0]), p(planes[1]), None, 0, None, 0, 3, hkv, d, PAGE, pages, here()))
    q = torch.randn(1, 16, d, generator=gen(25), device=DEV).to(BF)
    table, kv, out = ints([[pages - 1]]), ints([2]), torch.zeros(1, 16 * d, dtype=BF, device=DEV)
    ck(L, L.hbk_attn_paged_q4(p(q), 16 * d, p(planes[0]), p(planes[1]), p(table), 1, p(kv), None, p(out), 16 * d, None, 1, 1, 1, 64, 16, hkv, d, PAGE, 0, d ** -0.5, pages, 0, 0.0,
                              None, here()))
    torch.cuda.synchronize()
    last = [pl[-1:].clone() for pl in planes]
    want, mass = ref.attention(q, last[0], last[1], ints([[0]]), [2], [1], d ** -0.5)
    check_attn(out, want, mass, 16, d)
    c, s = ref.encode(x[2, :hkv * d].view(hkv, d // 32, 32))
    got_c, got_s = ref.plane_codes(planes[0][-2], d, True)
    assert torch.equal(got_c[:, 63], c.flatten(1)) and torch.equal(got_s[:, 63], s)


def test_calls_on_two_streams_at_once(L):
    """Different workspaces, the same cache and weights: neither disturbs the other."""
    hq, hkv, d = 32, 8, 128
    lens = [3000, 2000, 700, 64]
    kp, vp, table = cache(43, lens, hkv, d)
    w, vals = ref.q4_0_blocks(torch.randn(512, hq * d, generator=gen(44), device=DEV))
    packed = torch.zeros(L.hbk_gemm_q4_bytes(512, hq * d), dtype=torch.uint8, device=DEV)
    ck(L, L.hbk_gemm_q4_pack(p(w), p(packed), 512, hq * d, here()))
    qs = [torch.randn(4, hq, d, generator=gen(45 + i), device=DEV).to(BF) for i in range(2)]
    kv = ints(lens)
    n = L.hbk_attn_paged_q4_workspace_floats(4, 4, 1, 3000, hq, hkv, d, 0, 0)
    state = [(q, torch.empty(n, device=DEV), torch.zeros(4, hq * d, dtype=BF, device=DEV), torch.zeros(4, 512, device=DEV), torch.cuda.Stream()) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for q, work, o, y, s in state:
            ck(L, L.hbk_attn_paged_q4(p(q), hq * d, p(kp), p(vp), p(table), table.shape[1], p(kv), None, p(o), hq * d, p(work), 4, 4, 1, 3000, hq, hkv, d, PAGE, 0, d ** -0.5,
                                      kp.shape[0], 0, 0.0, None, s.cuda_stream))
            ck(L, L.hbk_gemm_q4(p(o), hq * d, p(packed), p(y), 512, None, 0, None, 4, 512, hq * d, 6, s.cuda_stream))
    torch.cuda.synchronize()
    for q, work, o, y, s in state:
        want, mass = ref.attention(q, kp, vp, table, lens, [1] * 4, d ** -0.5)
        check_attn(o, want, mass, hq, d)
        check_product(y, o, vals, 6)


def test_attention_large_and_small_numbers(L):
    """Scales of values from 2^-120 to 2^100 in different groups and growing along the sequence, queries from 2^-60 to 2^60 against keys that undo them."""
    hq, hkv, d, n = 4, 2, 128, 400
    pages = 7
    grow = torch.exp2(torch.linspace(-40, 40, pages * PAGE, device=DEV)).view(pages, 1, PAGE, 1)
    group = torch.exp2(torch.tensor([-70.0, -20.0, 0.0, 60.0], device=DEV)).repeat_interleave(32)
    v = torch.randn(pages, hkv, PAGE, d, generator=gen(8), device=DEV) * grow * group
    qs = torch.exp2(torch.tensor([60.0, -60.0], device=DEV)).view(1, 2, 1, 1)
    k = torch.randn(pages, hkv, PAGE, d, generator=gen(9), device=DEV) / qs
    kp, vp = ref.make_plane(k.to(BF), True), ref.make_plane(v.to(BF), False)
    q = (torch.randn(1, hkv, 2, d, generator=gen(10), device=DEV) * qs).view(1, hq, d).to(BF)
    table = torch.arange(pages, device=DEV).int()[None]
    want, mass = ref.attention(q, kp, vp, table, [n], [1], d ** -0.5)
    for split in (0, 1):
        check_attn(attn(L, q, kp, vp, table, [n], [1], d ** -0.5, split=split), want, mass, hq, d)
    # one query entry far above the others: those others count nothing in either
    q[0, 0, 3] = 2.0 ** 100
    q[0, 0, 4:] = 0
    kp[:, 0] = ref.make_plane(torch.where(torch.arange(d, device=DEV) == 3, 0.0, k[:, :1].double()).to(BF), True)[:, 0]
    want, mass = ref.attention(q, kp, vp, table, [n], [1], d ** -0.5)
    got = attn(L, q, kp, vp, table, [n], [1], d ** -0.5)
    assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("split", [0, 1])
def test_attention_keeps_infinities_and_nan_where_they_are_seen(L, split):
    hq, hkv, d = 4, 2, 128
    lens, rows = [200, 200, 200], [2, 1, 1]
    kp, vp, table = cache(31, lens, hkv, d)
    q = torch.randn(4, hq, d, generator=gen(12), device=DEV).to(BF)
    nan = torch.tensor([0xFF, 0xFF], dtype=torch.uint8, device=DEV)

    def scale_at(plane, b, pos, h, group):
        page = int(table[b, pos // PAGE])
        return plane[page, h, PAGE * d // 2 + ((pos % PAGE) * 4 + group) * 2:][:2]

    scale_at(vp, 0, 199, 0, 1)[:] = nan      # the last position: row 0 of sequence 0 does not see it, row 1 does
    scale_at(kp, 1, 50, 1, 2)[:] = nan       # a key: the whole of heads 2, 3
    out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split).view(4, hq, d)
    want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.isnan(out[1, :2, 32:64]).all() and not torch.isnan(out[0]).any() and torch.isnan(out[2, 2:]).all()
    fine = ~torch.isnan(want)
    check_attn(torch.where(fine, out.double(), 0.0).flatten(1), torch.where(fine, want, 0.0), torch.where(fine, mass, 0.0), hq, d)
    # outside a window neither is seen
    out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, window=100, split=split).view(4, hq, d)
    assert not torch.isnan(out[2:]).any()
    q[3, 1] = float("nan")
    q[3, 2, 5] = float("inf")
    out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split).view(4, hq, d)
    assert torch.isnan(out[3, 1:3]).all() and not torch.isnan(out[3, 0]).any() and not torch.isnan(out[3, 3]).any()


def test_attention_does_not_see_pages_that_are_none(L):
    hq, hkv, d = 4, 2, 64
    lens = [500, 500]
    kp, vp, table = cache(37, lens, hkv, d)
    table[0, 2], table[0, 5], table[1, 0] = -1, kp.shape[0], 2 ** 31 - 1
    q = torch.randn(2, hq, d, generator=gen(13), device=DEV).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, [1, 1], d ** -0.5)
    for split in (0, 1, 4):
        check_attn(attn(L, q, kp, vp, table, lens, [1, 1], d ** -0.5, split=split), want, mass, hq, d)
    table[:] = -1
    assert (attn(L, q, kp, vp, table, lens, [1, 1], d ** -0.5) == 0).all()


def test_attention_cuts_what_lies_past_the_bounds(L):
    """Lengths above max_kv_len or the table's width: no read past either."""
    hq, hkv, d = 4, 2, 128
    kp, vp, table = cache(41, [300, 300], hkv, d)
    q = torch.randn(2, hq, d, generator=gen(14), device=DEV).to(BF)
    want, mass = ref.attention(q, kp, vp, table, [256, 128], [1, 1], d ** -0.5)
    out = attn(L, q, kp, vp, table[:, :4].contiguous(), [10 ** 6, 128], [1, 1], d ** -0.5, longest_kv=256)
    check_attn(out, want, mass, hq, d)


@pytest.mark.parametrize("window,softcap,sink", [(0, 0.0, False), (1, 0.0, True), (70, 30.0, False), (300, 0.0, True), (0, 5.0, True)])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (9, 1, 64)])
def test_portions_of_many_columns(L, hq, hkv, d, window, softcap, sink):
    """256 columns and more per kv head: whole prompts, a prefix, one token, nothing, more rows than positions; rows of no sequence stay."""
    lens, rows = [64, 700, 130, 0, 257, 65], [64, 64, 1, 0, 40, 33]
    kp, vp, table = cache(d + window, lens, hkv, d)
    T = sum(rows)
    q = (2 * torch.randn(T + 3, hq, d, generator=gen(2), device=DEV)).to(BF)
    sk = torch.randn(hq, generator=gen(3), device=DEV).to(BF) * 3 if sink else None
    want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5, window, softcap, sk)
    for split in (0, 1, 3):
        out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, window, softcap, sk, split=split, ldo=hq * d + (1 if split == 1 else 8))
        check_attn(out[:T], want[:T], mass[:T], hq, d)
        assert (out[T:] == 9).all() and (out[:, hq * d:] == 9).all()
    out = attn(L, q[:100], kp, vp, table, [60], [100], d ** -0.5)  # its first 40 rows see nothing
    want, mass = ref.attention(q[40:100], kp, vp, table, [60], [60], d ** -0.5)
    assert (out[:40] == 0).all()
    check_attn(out[40:], want, mass, hq, d)


@pytest.mark.parametrize("scale", [-0.125, 0.0, 3e-30, 2.0])
def test_portions_of_many_columns_scales(L, scale):
    hq, hkv, d, lens, rows = 8, 1, 128, [300, 65], [40, 33]
    kp, vp, table = cache(3, lens, hkv, d)
    q = torch.randn(sum(rows), hq, d, generator=gen(21), device=DEV).to(BF)
    for window, cap in ((0, 0.0), (2 ** 31 - 1, 0.0), (70, 20.0)):
        want, mass = ref.attention(q, kp, vp, table, lens, rows, scale, window, cap)
        for split in (0, 1):
            check_attn(attn(L, q, kp, vp, table, lens, rows, scale, window, cap, split=split), want, mass, hq, d)


def test_portions_of_many_columns_large_and_small_numbers(L):
    """Value scales from 2^-120 to 2^100 in different groups, growing along the sequence; keys of 2^-60 and 2^60 under queries that undo them."""
    hq, hkv, d, n, r = 16, 2, 128, 400, 40
    pages = 7
    grow = torch.exp2(torch.linspace(-40, 40, pages * PAGE, device=DEV)).view(pages, 1, PAGE, 1)
    group = torch.exp2(torch.tensor([-70.0, -20.0, 0.0, 60.0], device=DEV)).repeat_interleave(32)
    v = torch.randn(pages, hkv, PAGE, d, generator=gen(8), device=DEV) * grow * group
    qs = torch.exp2(torch.tensor([60.0, -60.0], device=DEV)).view(1, 2, 1, 1)
    k = torch.randn(pages, hkv, PAGE, d, generator=gen(9), device=DEV) / qs
    kp, vp = ref.make_plane(k.to(BF), True), ref.make_plane(v.to(BF), False)
    q = (torch.randn(r, hkv, hq // hkv, d, generator=gen(10), device=DEV) * qs).view(r, hq, d).to(BF)
    table = torch.arange(pages, device=DEV).int()[None]
    want, mass = ref.attention(q, kp, vp, table, [n], [r], d ** -0.5)
    for split in (0, 1):
        check_attn(attn(L, q, kp, vp, table, [n], [r], d ** -0.5, split=split), want, mass, hq, d)


@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_portions_of_many_columns_keep_infinities_and_nan_where_they_are_seen(L, d, split):
    hq, hkv, J = 16, 2, d // 32
    lens, rows = [200, 200, 150], [40, 40, 33]
    kp, vp, table = cache(31, lens, hkv, d)
    q = torch.randn(sum(rows), hq, d, generator=gen(12), device=DEV).to(BF)

    def scale_at(plane, b, pos, h, group, value):
        s = plane[int(table[b, pos // PAGE]), h, PAGE * d // 2 + ((pos % PAGE) * J + group) * 2:][:2]
        s[:] = torch.tensor([value], dtype=BF).view(torch.uint8).to(DEV)

    scale_at(vp, 0, 180, 0, 1, float("nan"))   # seen by the rows from 180 on
    scale_at(vp, 0, 199, 1, 0, float("inf"))   # by the last
    scale_at(vp, 0, 170, 1, 1, float("-inf"))
    scale_at(vp, 1, 20, 0, 0, float("inf"))    # by all
    scale_at(kp, 1, 50, 1, 1, float("nan"))    # by all: the whole of these heads
    scale_at(kp, 2, 140, 0, 0, float("nan"))   # by the rows from 140 on
    for window in (0, 25):
        want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5, window)
        out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, window, split=split).view(-1, hq, d)
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~fine & ~torch.isnan(want)].double(), want[~fine & ~torch.isnan(want)])
        assert fine[9].all() and fine[19, :8].all() and not fine[20:40, :8, 32:64].any() and not fine[39, 8:, :32].any()  # (of the plain result)
        check_attn(torch.where(fine, out.double(), 0.0).flatten(1), torch.where(fine, want, 0.0), torch.where(fine, mass, 0.0), hq, d)


def test_portions_of_many_columns_queries_that_are_none(L):
    """A NaN or an infinity in a query is its own column's matter."""
    hq, hkv, d, lens, rows = 16, 2, 128, [200], [40]
    kp, vp, table = cache(33, lens, hkv, d)
    q = torch.randn(40, hq, d, generator=gen(16), device=DEV).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5)
    q[3, 5, 17], q[39, 15, 0] = float("nan"), float("inf")
    for split in (0, 1):
        out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split).view(-1, hq, d)
        assert torch.isnan(out[3, 5]).all() and torch.isnan(out[39, 15]).all()
        out[3, 5], out[39, 15] = want[3, 5].to(BF), want[39, 15].to(BF)
        check_attn(out.flatten(1), want, mass, hq, d)


def test_portions_of_many_columns_do_not_see_pages_that_are_none(L):
    hq, hkv, d, rows = 8, 1, 128, [40, 33]
    lens = [500, 200]
    kp, vp, table = cache(37, lens, hkv, d)
    table[0, 0], table[0, 2], table[0, 7], table[1, 1] = -1, kp.shape[0], 2 ** 31 - 1, -5
    q = torch.randn(sum(rows), hq, d, generator=gen(13), device=DEV).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5)
    for split in (0, 1, 4):
        check_attn(attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split), want, mass, hq, d)
    table[:] = -1
    for split in (0, 1):
        assert (attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split) == 0).all()


def test_portions_of_many_columns_bits_depend_on_the_sequence_and_the_split_alone(L):
    hq, hkv, d = 32, 4, 128
    lens, rows = [1500, 40, 777, 3000, 0], [64, 40, 5, 33, 0]
    kp, vp, table = cache(23, lens, hkv, d)
    q = torch.randn(sum(rows), hq, d, generator=gen(6), device=DEV).to(BF)
    full = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=8, longest_kv=50000)
    for b in range(4):
        at = slice(sum(rows[:b]), sum(rows[:b + 1]))
        assert torch.equal(full[at], attn(L, q[at], kp, vp, table[b:b + 1].clone(), lens[b:b + 1], rows[b:b + 1], d ** -0.5, split=8, most=64))
    assert torch.equal(full, attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=8, longest_kv=50000))


@pytest.mark.parametrize("hq,d", [(256, 64), (300, 128)])
def test_single_tokens_of_many_heads_per_kv_head(L, hq, d):
    lens = [1, 63, 64, 0, 65, 700]
    kp, vp, table = cache(29, lens, 1, d)
    q = torch.randn(len(lens), hq, d, generator=gen(15), device=DEV).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, [1] * 6, d ** -0.5)
    for split in (0, 2):
        for cu in (True, False):
            check_attn(attn(L, q, kp, vp, table, lens, [1] * 6, d ** -0.5, split=split, cu=cu), want, mass, hq, d)


def test_portions_of_many_columns_over_a_long_cache(L):
    hq, hkv, d, lens, rows = 8, 1, 64, [40000, 64, 9000], [33, 64, 1]
    kp, vp, table = cache(17, lens, hkv, d, spread=0.3, width=700)
    q = (1.5 * torch.randn(sum(rows), hq, d, generator=gen(5), device=DEV)).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, rows, d ** -0.5)
    for split in (0, 64, 1000):
        check_attn(attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split), want, mass, hq, d)


def test_portions_of_many_columns_captured_on_two_streams(L):
    """Two calls at once, each captured and replayed: the same bits as by itself."""
    hq, hkv, d, rows, lens = 16, 2, 128, [64, 40], [900, 300]
    kp, vp, table = cache(51, lens, hkv, d)
    calls = []
    for i in range(2):
        q = torch.randn(sum(rows), hq, d, generator=gen(70 + i), device=DEV).to(BF)
        want = attn(L, q, kp, vp, table, lens, rows, d ** -0.5)
        n = L.hbk_attn_paged_q4_workspace_floats(2, sum(rows), 64, 900, hq, hkv, d, 0, 0)
        args = dict(q=q, out=torch.zeros_like(want), work=torch.empty(max(n, 4), device=DEV), cu=ints([0, 64, 104]), kv=ints(lens))
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ck(L, L.hbk_attn_paged_q4(p(q), hq * d, p(kp), p(vp), p(table), table.shape[1], p(args["kv"]), p(args["cu"]), p(args["out"]), hq * d, p(args["work"]),
                                      2, sum(rows), 64, 900, hq, hkv, d, PAGE, 0, d ** -0.5, kp.shape[0], 0, 0.0, None, stream.cuda_stream))
        calls.append((args, want, stream, graph))
    for _ in range(20):
        for args, _, stream, graph in calls:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for args, want, _, _ in calls:
        assert torch.equal(args["out"], want)


# (columns of a tile: up to 8, up to 16, 128)
TILES = [(2, 1, 3), (4, 1, 4), (9, 3, 5), (8, 1, 40)]


@pytest.mark.parametrize("up", [2, 12, 16, 17, 22, 26, 30, 100])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,rows", TILES)
def test_attention_values_that_a_row_does_not_see_have_no_part_in_it(L, hq, hkv, rows, d, up):
    """The last position's values are 2^up times the others' in one group: the rows before it see nothing of them."""
    n = 200
    k, v = (torch.randn(4, hkv, PAGE, d, generator=gen(80 + i), device=DEV) for i in range(2))
    v[(n - 1) // PAGE, :, (n - 1) % PAGE, 32:64] *= 2.0 ** up
    kp, vp = ref.make_plane(k.to(BF), True), ref.make_plane(v.to(BF), False)
    q = torch.randn(rows, hq, d, generator=gen(82), device=DEV).to(BF)
    table = torch.arange(4, device=DEV).int()[None]
    want, mass = ref.attention(q, kp, vp, table, [n], [rows], d ** -0.5)
    for split in (0, 1):
        check_attn(attn(L, q, kp, vp, table, [n], [rows], d ** -0.5, split=split), want, mass, hq, d)


@pytest.mark.parametrize("up", [10, 16, 17, 22, 30, 60])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,rows", [(1, 1, 1)] + TILES)
def test_attention_large_values_of_no_weight_leave_the_others_as_they_are(L, hq, hkv, rows, d, up):
    """One position's values are 2^up times the others', its weight e^-180 of theirs: every row sees it, and it counts next to nothing."""
    n, at = 200, 70
    base = torch.randn(hkv, 1, d, generator=gen(83), device=DEV)
    q = (base + 0.1 * torch.randn(rows, hkv, hq // hkv, d, generator=gen(84), device=DEV)).view(rows, hq, d).to(BF)
    k, v = (torch.randn(4, hkv, PAGE, d, generator=gen(85 + i), device=DEV) for i in range(2))
    k[at // PAGE, :, at % PAGE] = -180 * base[:, 0] * d ** 0.5 / base[:, 0].square().sum(-1, keepdim=True)
    kp, small = ref.make_plane(k.to(BF), True), ref.make_plane(v.to(BF), False)
    v[at // PAGE, :, at % PAGE, :32] *= 2.0 ** up
    vp = ref.make_plane(v.to(BF), False)
    table = torch.arange(4, device=DEV).int()[None]
    want, _ = ref.attention(q, kp, vp, table, [n], [rows], d ** -0.5)
    other, mass = ref.attention(q, kp, small, table, [n], [rows], d ** -0.5)
    assert torch.allclose(want, other, rtol=1e-12, atol=1e-12)  # (of the plain results)
    for split in (0, 1):
        check_attn(attn(L, q, kp, vp, table, [n], [rows], d ** -0.5, split=split), want, mass, hq, d)


def mass_of(monkeypatch, *args):
    """Sum of p |v|, nothing more: what a result's error goes by where values are far apart."""
    real = ref.plane_values
    with monkeypatch.context() as m:
        m.setattr(ref, "plane_values", lambda plane, d, keys: real(plane, d, keys) if keys else real(plane, d, keys).abs())
        return ref.attention(*args)[0]


@pytest.mark.parametrize("window,softcap,sink", [(0, 0.0, False), (70, 0.0, True), (0, 20.0, True), (1, 30.0, False)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (24, 2, 64)])
@pytest.mark.parametrize("most", [1, 9, 140])
def test_attention_of_values_far_apart(L, monkeypatch, hq, hkv, d, window, softcap, sink, most):
    """Value scales from 2^-60 to 2^60 in no order: pages that are none, lengths of zero and one, more shares than one."""
    lens = [1, 65, 130, 0, 700, 257, 64]
    rows = [min(n, most) if i != 1 else 1 for i, n in enumerate(lens)]
    kp, vp, table = cache(d + window, lens, hkv, d, spread=20.0)
    table[4, 3], table[5, 0] = -1, kp.shape[0]
    q = torch.randn(sum(rows) + 2, hq, d, generator=gen(86), device=DEV).to(BF)
    sk = torch.randn(hq, generator=gen(87), device=DEV).to(BF) * 3 if sink else None
    args = (q, kp, vp, table, lens, rows, d ** -0.5, window, softcap, sk)
    want, mass = ref.attention(*args)[0], mass_of(monkeypatch, *args)
    for split in (0, 1, 3):
        out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, window, softcap, sk, split=split, ldo=hq * d + 8)
        check_attn(out[:-2], want[:-2], mass[:-2], hq, d)
        assert (out[-2:] == 9).all() and (out[:, hq * d:] == 9).all()


@pytest.mark.parametrize("hq,hkv,rows", TILES)
def test_attention_of_values_far_apart_keeps_infinities_and_nan_where_they_are_seen(L, monkeypatch, hq, hkv, rows):
    d, lens = 128, [200, 200]
    kp, vp, table = cache(88, lens, hkv, d, spread=20.0)
    q = torch.randn(2 * rows, hq, d, generator=gen(89), device=DEV).to(BF)

    def scale_at(plane, b, pos, h, group, value):
        plane[int(table[b, pos // PAGE]), h, PAGE * d // 2 + ((pos % PAGE) * 4 + group) * 2:][:2] = torch.tensor([value], dtype=BF).view(torch.uint8).to(DEV)

    scale_at(vp, 0, 199, 0, 1, float("nan"))
    scale_at(vp, 0, 198, 0, 3, float("inf"))
    scale_at(kp, 1, 199, hkv - 1, 2, float("nan"))
    args = (q, kp, vp, table, lens, [rows, rows], d ** -0.5)
    want, mass = ref.attention(*args)[0], mass_of(monkeypatch, *args)
    fine = torch.isfinite(want)
    assert fine[:rows - 2].all() and not fine[rows - 1, 0, 32:64].any() and fine[rows:2 * rows - 1].all()  # (of the plain result)
    for split in (0, 1):
        out = attn(L, q, kp, vp, table, lens, [rows, rows], d ** -0.5, split=split).view(-1, hq, d)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~fine & ~torch.isnan(want)].double(), want[~fine & ~torch.isnan(want)])
        check_attn(torch.where(fine, out.double(), 0.0).flatten(1), torch.where(fine, want, 0.0), torch.where(fine, mass, 0.0), hq, d)


@pytest.mark.parametrize("softcap", [1e-39, 1e-30, 0.01, 60.0, 70.0, 300.0, 1e4, 1e7, 1e30, 3e38])
@pytest.mark.parametrize("hq,hkv,rows", [(1, 1, 1)] + TILES)
def test_attention_caps_of_any_size(L, hq, hkv, rows, softcap):
    """Scores to some 60 on either side: a cap far above leaves them as they are, one far below makes all positions alike."""
    d, lens = 64, [300, 65]
    softcap = float(torch.tensor(softcap, dtype=torch.float32))
    kp, vp, table = cache(90, lens, hkv, d)
    q = (15 * torch.randn(2 * rows, hq, d, generator=gen(91), device=DEV)).to(BF)
    want, mass = ref.attention(q, kp, vp, table, lens, [rows, rows], d ** -0.5, 0, softcap)
    for split in (0, 1):
        check_attn(attn(L, q, kp, vp, table, lens, [rows, rows], d ** -0.5, 0, softcap, split=split), want, mass, hq, d)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("split", [3, 100])
def test_waits_that_run_out_end_the_call_and_are_said(L, d, split):
    """A limit so short that the waits inside the kernel are given up: its rows are NaN, the status says so once, and the calls that follow are right."""
    hq, hkv, lens, rows = 16, 2, [900, 64, 300], [64, 40, 1]
    kp, vp, table = cache(92, lens, hkv, d)
    T = sum(rows)
    q = torch.randn(T + 2, hq, d, generator=gen(93), device=DEV).to(BF)
    good = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split)
    assert L.hbk_attn_paged_q4_status() == 0
    former = L.hbk_attn_paged_q4_wait_cycles(-1)
    try:
        out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split)
        assert torch.isnan(out[:T]).all() and (out[T:] == 9).all()
        assert L.hbk_attn_paged_q4_status() == 702 and b"timed out" in L.hbk_last_error()
        assert L.hbk_attn_paged_q4_status() == 0
        for cycles in (0, 500, 2000, 8000):  # some waits go well
            L.hbk_attn_paged_q4_wait_cycles(cycles)
            out = attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split)
            void = torch.isnan(out)
            assert torch.equal(torch.where(void, 0, out), torch.where(void, 0, good)) and L.hbk_attn_paged_q4_status() == (702 if void.any() else 0)
    finally:
        L.hbk_attn_paged_q4_wait_cycles(former)
    assert torch.equal(attn(L, q, kp, vp, table, lens, rows, d ** -0.5, split=split), good) and L.hbk_attn_paged_q4_status() == 0


@pytest.mark.parametrize("hkv,rows,most", [(8192, 150, 200), (16400, 400, 600)])
def test_attention_of_more_tiles_and_heads_than_a_launch_has_room_for(L, hkv, rows, most):
    """Tiles times kv heads above 65535, with 16 and with 128 columns per tile: a few of the heads in 64 bits, and with the bits that they have by themselves."""
    d, n = 64, rows + 30
    pages = -(-n // PAGE)
    kp, vp = (torch.randint(0, 256, (pages, hkv, PAGE * d // 2 + PAGE * d // 16), generator=gen(94 + i), device=DEV, dtype=torch.uint8) for i in range(2))
    for plane in (kp, vp):
        plane[..., PAGE * d // 2:] = (0.2 * torch.randn(pages, hkv, PAGE * d // 32, generator=gen(96), device=DEV)).to(BF).view(torch.uint8)
    q = torch.randn(rows, hkv, d, generator=gen(97), device=DEV, dtype=BF)
    table = torch.randperm(pages, generator=gen(98), device=DEV).int()[None]
    for split in (3, 100):
        out = attn(L, q, kp, vp, table, [n], [rows], d ** -0.5, split=split, most=most).view(rows, hkv, d)
        for h in (0, hkv // 3, hkv - 1):
            one = [x[:, h:h + 1].contiguous() for x in (q, kp, vp)]
            got = out[:, h].contiguous()
            check_attn(got, *ref.attention(*one, table, [n], [rows], d ** -0.5), 1, d)
            assert torch.equal(got, attn(L, *one, table, [n], [rows], d ** -0.5, split=split, most=most))


@pytest.mark.parametrize("hq,hkv,rows", TILES)
@pytest.mark.parametrize("up", [2.0 ** 100, 2.0 ** -100])
def test_attention_one_query_entry_far_above_the_others(L, hq, hkv, rows, up):
    """Against keys that are 0 there it adds nothing, against others it decides: results, not only that they are finite."""
    d, lens = 128, [400, 70]
    k, v = (torch.randn(10, hkv, PAGE, d, generator=gen(100 + i), device=DEV) for i in range(2))
    q = torch.randn(2 * rows, hq, d, generator=gen(102), device=DEV) * up
    q[:, 0], q[:, 0, 3] = 0, up
    k[:, 0, :, 3] = 0
    k /= up
    k[5:, :, :, 3] = 0.25 / up  # of the second sequence
    kp, vp = ref.make_plane(k.to(BF), True), ref.make_plane(v.to(BF), False)
    q = q.to(BF)
    table = ints([[0, 1, 2, 3, 4, 9, 8], [5, 6, -1, -1, -1, -1, -1]])
    want, mass = ref.attention(q, kp, vp, table, lens, [rows, rows], d ** -0.5)
    for split in (0, 1):
        check_attn(attn(L, q, kp, vp, table, lens, [rows, rows], d ** -0.5, split=split), want, mass, hq, d)


# ------------------------------------------------------------------ products
def product(L, x, w, N, K, epi, out=None, r=None, bias=None, pack=True):
    M = x.shape[0]
    n = L.hbk_gemm_q4_bytes(N, K)
    packed = torch.full((n + 16,), 0xEE, dtype=torch.uint8, device=DEV)
    ck(L, L.hbk_gemm_q4_pack(p(w), p(packed), N, K, here()))
    out = torch.full((M + 1, N + 3), 9.0, dtype=torch.float32 if epi == 6 else BF, device=DEV) if out is None else out
    ck(L, L.hbk_gemm_q4(p(x), x.stride(0), p(packed), p(out), out.stride(0), p(r), r.stride(0) if r is not None else 0, p(bias), M, N, K, epi, here()))
    torch.cuda.synchronize()
    assert (packed[n:] == 0xEE).all()
    return out


def check_product(got, x, w, epi, r=None, bias=None):
    """fp32 sums: of K / 32 groups and their products, at most K / 32 + 40 roundings of 2^-24 (and truncations of 2^-23) of the sum of |x w|; the
    result's own rounding to bf16 (2^-8)."""
    want, mass = x.double() @ w.T, x.double().abs() @ w.abs().T
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    if r is not None:
        want, mass = want + r.double(), mass + r.double().abs()
    tol = mass * (x.shape[1] / 32 + 40) * 2.0 ** -23 + 1e-30
    if epi != 6:
        tol = tol + 2.0 ** -8 * want.abs()
    off = (got.double() - want).abs() - tol
    assert (off <= 0).all(), off.max().item()
    if epi == 6:  # and on the whole far less: roundings do not add up
        assert (got.double() - want).norm() <= 2e-6 * want.norm()


@pytest.mark.parametrize("epi", [0, 1, 3, 4, 6])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 16, 128), (2, 17, 96), (5, 130, 4096), (7, 1000, 160), (8, 64, 2048), (9, 33, 416), (13, 515, 1056), (16, 4096, 512),
                                   (17, 40, 128), (31, 100, 8960), (32, 2048, 256), (33, 48, 320), (64, 96, 1024), (100, 70, 544), (256, 50, 96)])
def test_product(L, M, N, K, epi):
    w, vals = ref.q4_0_blocks(torch.randn(N, K, generator=gen(N), device=DEV) * K ** -0.5)
    x = torch.randn(M, K + 8, generator=gen(K), device=DEV).to(BF)[:, :K]
    bias = torch.randn(N, generator=gen(1), device=DEV).to(BF) if epi in (1, 4) else None
    r = torch.randn(M, N + 5, generator=gen(2), device=DEV).to(BF)[:, :N] if epi in (3, 4) else None
    out = product(L, x, w, N, K, epi, r=r, bias=bias)
    check_product(out[:M, :N], x, vals, epi, r, bias)
    assert (out[M] == 9).all() and (out[:, N:] == 9).all()


def test_product_residual_in_place_and_again(L):
    M, N, K = 6, 300, 1024
    w, vals = ref.q4_0_blocks(torch.randn(N, K, generator=gen(3), device=DEV))
    x = torch.randn(M, K, generator=gen(4), device=DEV).to(BF)
    r = torch.randn(M, N, generator=gen(5), device=DEV).to(BF)
    out = r.clone()
    product(L, x, w, N, K, 3, out=out, r=out)
    check_product(out, x, vals, 3, r)
    a, b = product(L, x, w, N, K, 6), product(L, x, w, N, K, 6)
    assert torch.equal(a, b)


def test_product_of_any_bytes(L):
    """Random blocks: all codes, scales of both signs, subnormal ones, zero."""
    M, N, K = 4, 200, 1280
    c = torch.randint(0, 16, (N, K // 32, 32), generator=gen(6), device=DEV)
    s = torch.randn(N, K // 32, generator=gen(7), device=DEV).to(torch.float16)
    s[::3] *= 2.0 ** -14
    s[::7] = 6e-8
    s[::11] = 0
    x = torch.randn(M, K, generator=gen(8), device=DEV).to(BF)
    out = product(L, x, ref.blocks_of(c, s), N, K, 6)
    check_product(out[:M, :N], x, ((c - 8).double() * s.double()[..., None]).flatten(1), 0)


def test_product_keeps_infinities_and_nan_in_their_rows(L):
    M, N, K = 9, 64, 256
    w, vals = ref.q4_0_blocks(torch.randn(N, K, generator=gen(9), device=DEV))
    x = torch.randn(M, K, generator=gen(10), device=DEV).to(BF)
    x[2, 7], x[8, 200] = float("nan"), float("inf")
    out = product(L, x, w, N, K, 6)[:M, :N]
    fine = [i for i in range(M) if i not in (2, 8)]
    check_product(out[fine], x[fine], vals, 6)
    assert torch.isnan(out[2]).all() and not torch.isfinite(out[8]).any()
    want = torch.where(vals[:, 200] == 0, float("nan"), torch.sign(vals[:, 200]) * float("inf")).float()
    assert torch.equal(torch.nan_to_num(out[8], nan=1.0), torch.nan_to_num(want, nan=1.0))


@pytest.mark.parametrize("M", [1, 4, 13, 32])
def test_product_of_any_bytes_in_fp32(L, M):
    """Random blocks, a result in fp32: its own rounding hides nothing."""
    N, K = 200, 1280
    c = torch.randint(0, 16, (N, K // 32, 32), generator=gen(106), device=DEV)
    s = torch.randn(N, K // 32, generator=gen(107), device=DEV).to(torch.float16)
    s[::3] *= 2.0 ** -14
    s[::7] = 6e-8
    s[::11] = 0
    x = torch.randn(M, K, generator=gen(108), device=DEV).to(BF)
    out = product(L, x, ref.blocks_of(c, s), N, K, 6)[:M, :N]
    w = ((c - 8).double() * s.double()[..., None]).flatten(1)
    check_product(out, x, w, 6)
    for rows in (slice(0, None, 3), slice(0, None, 7)):  # the small ones by themselves
        check_product(out[:, rows], x, w[rows], 6)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 3, 64)])
def test_steps_together_captured_and_replayed(L, hq, hkv, d):
    """Tables, write, attention, output projection of several decode steps in one captured graph on a stream of its own, replayed; then
    the same by hand in 64 bits."""
    B, width, pages, steps, hidden = 5, 6, 24, 130, 96
    state = dict(ctx=[0, 5, 63, 64, 100])
    held = [-(-c // PAGE) for c in state["ctx"]]
    ids = list(range(pages))[::-1]
    table = [[ids.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    tb, fr, count, ctx, new = ints(table), ints(ids + [-1] * (pages - len(ids))), ints([len(ids)]), ints(state["ctx"]), ints([1, 1, 1, 1, 1])
    cu, pos, slot = ints([0] * (B + 1)), ints([0] * B), ints([0] * B)
    planes = [ref.make_plane(torch.randn(pages, hkv, PAGE, d, generator=gen(50 + i), device=DEV).to(BF), i == 0) for i in range(2)]
    start = [x.clone() for x in planes]
    qkv = torch.zeros(B, (hq + 2 * hkv) * d, dtype=BF, device=DEV)
    rows = torch.randn(steps, B, (hq + 2 * hkv) * d, generator=gen(60), device=DEV).to(BF)
    w, vals = ref.q4_0_blocks(torch.randn(hidden, hq * d, generator=gen(61), device=DEV))
    packed = torch.zeros(L.hbk_gemm_q4_bytes(hidden, hq * d), dtype=torch.uint8, device=DEV)
    ck(L, L.hbk_gemm_q4_pack(p(w), p(packed), hidden, hq * d, here()))
    o, y = torch.zeros(B, hq * d, dtype=BF, device=DEV), torch.zeros(B, hidden, device=DEV)
    n = L.hbk_attn_paged_q4_workspace_floats(B, B, 1, width * PAGE, hq, hkv, d, 2, 0)
    work = torch.empty(n, device=DEV)
    ld = qkv.shape[1]
    torch.cuda.synchronize()

    def step(stream):
        k, v = qkv[:, hq * d:], qkv[:, (hq + hkv) * d:]
        ck(L, L.hbk_page_tables(p(ctx), p(new), B, p(tb), width, p(fr), p(count), p(count), pages, p(cu), p(ctx), p(pos), p(slot), B, PAGE, stream))
        ck(L, L.hbk_kv_write_q4(p(k), ld, p(v), ld, p(slot), p(planes[0]), p(planes[1]), None, 0, None, 0, B, hkv, d, PAGE, pages, stream))
        ck(L, L.hbk_attn_paged_q4(p(qkv), ld, p(planes[0]), p(planes[1]), p(tb), width, p(ctx), p(cu), p(o), hq * d, p(work), B, B, 1, width * PAGE, hq, hkv, d,
                                  PAGE, 2, d ** -0.5, pages, 0, 0.0, None, stream))
        ck(L, L.hbk_gemm_q4(p(o), hq * d, p(packed), p(y), hidden, None, 0, None, B, hidden, hq * d, 6, stream))

    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(here())
    lens = list(state["ctx"])
    for i in range(steps):
        qkv.copy_(rows[i])
        graph.replay()
        lens = [c + 1 for c in lens]
        if i in (0, 1, 63, 64, steps - 1):
            torch.cuda.synchronize()
            assert ctx.tolist() == lens and cu.tolist() == list(range(B + 1)) and pos.tolist() == [c - 1 for c in lens]
            want, mass = ref.attention(rows[i, :, :hq * d].view(B, hq, d), planes[0], planes[1], tb, lens, [1] * B, d ** -0.5)
            check_attn(o, want, mass, hq, d)
            check_product(y, o, vals, 6)
    # the cache holds what was written, at the places that the tables say, and nothing else has changed
    k0 = rows[:, :, hq * d:(hq + hkv) * d].reshape(steps, B, hkv, d)
    for b in range(B):
        for i in (0, 1, 62, 63, steps - 1):
            at = state["ctx"][b] + i
            c, sc = ref.encode(k0[i, b].unflatten(-1, (-1, 32)))
            got_c, got_s = ref.plane_codes(planes[0][int(tb[b, at // PAGE])], d, True)
            assert torch.equal(got_c[:, at % PAGE], c.flatten(-2)) and torch.equal(got_s[:, at % PAGE], sc)
    first = int(tb[4, 0])
    for was, now in zip(start, planes):
        assert torch.equal(was[first], now[first])
    used = sum(-(-c // PAGE) for c in lens)
    assert count.item() == pages - used
