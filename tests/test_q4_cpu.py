"""The calls of the 4-bit step that are refused, and their host arithmetic (no GPU: nothing is launched)."""
import ctypes as C

import pytest

import helix_b200 as hb

L = hb.load_library()
OK = 4096  # an address that is aligned; refused calls never look at it


def tables(B=4, max_pages=8, num_pages=100, T=4, page=64, null=None):
    ptr = [None if null == i else OK for i in range(10)]
    return L.hbk_page_tables(ptr[0], ptr[1], B, ptr[2], max_pages, ptr[3], ptr[4], ptr[5], num_pages, ptr[6], ptr[7], ptr[8], ptr[9], T, page, None)


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=-1), dict(B=2049), dict(max_pages=0), dict(max_pages=2 ** 31 - 1), dict(num_pages=0), dict(num_pages=2 ** 26), dict(T=-1),
                                dict(page=32)] + [dict(null=i) for i in range(10)])
def test_page_tables_refusals(kw):
    assert tables(**kw) == 1 and b"invalid argument" in L.hbk_last_error()


def test_page_tables_rows_that_indices_do_not_reach():
    assert tables(T=2 ** 30 + 1) == 1 and tables(T=2 ** 31 - 1) == 1


@pytest.mark.parametrize("N,K", [(16, 2 ** 30), (16, 2 ** 31 - 32), (65535 * 64 + 1, 32), (2 ** 31 - 1, 128)])
def test_weights_beyond_the_products_sizes(N, K):
    """Refused by the size, the packing and the product alike."""
    assert L.hbk_gemm_q4_bytes(N, K) == 0 and L.hbk_gemm_q4_pack(OK, OK, N, K, None) == 1 and gemm(N=N, K=K, ldx=2 ** 31 - 8, ldo=2 ** 31 - 1) == 1
    assert L.hbk_gemm_q4_bytes(65535 * 64, 128) == 65535 * 64 * 72 and L.hbk_gemm_q4_bytes(16, 2 ** 30 - 128) == (2 ** 30 - 128) * 9


def write(k=OK, ldk=256, v=OK, ldv=256, slots=OK, kc=OK, vc=OK, ks=None, ldks=0, vs=None, ldvs=0, T=3, hkv=2, d=128, page=64, pages=10):
    return L.hbk_kv_write_q4(k, ldk, v, ldv, slots, kc, vc, ks, ldks, vs, ldvs, T, hkv, d, page, pages, None)


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(k=OK + 2), dict(v=OK + 8), dict(kc=OK + 4), dict(vc=OK + 8),
                                dict(ldk=248), dict(ldv=260), dict(ldk=0), dict(ks=OK, ldks=8), dict(vs=OK + 2, ldvs=256), dict(T=-1), dict(hkv=0), dict(d=96), dict(d=256),
                                dict(page=16), dict(pages=0), dict(pages=2 ** 26), dict(hkv=65536, ldk=2 ** 23, ldv=2 ** 23)])
def test_kv_write_refusals(kw):
    assert write(**kw) == 1


def test_nothing_to_do_is_no_error():
    assert write(T=0) == 0 and attn(T=0) == 0 and gemm(M=0) == 0


def attn(q=OK, ldq=1024, kc=OK, vc=OK, table=OK, max_pages=8, kv=OK, cu=OK, out=OK, ldo=1024, work=OK, B=4, T=4, most=1, longest=512, hq=8, hkv=2, d=128, page=64,
         split=4, scale=0.1, pages=100, window=0, cap=0.0, sink=None):
    return L.hbk_attn_paged_q4(q, ldq, kc, vc, table, max_pages, kv, cu, out, ldo, work, B, T, most, longest, hq, hkv, d, page, split, scale, pages, window, cap, sink, None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(kc=None), dict(vc=None), dict(table=None), dict(kv=None), dict(out=None), dict(work=None), dict(q=OK + 2), dict(kc=OK + 8),
                                dict(vc=OK + 2), dict(ldq=1016), dict(ldq=1028), dict(ldo=1016), dict(out=OK + 1), dict(B=0), dict(B=65536), dict(T=-1), dict(most=0), dict(longest=-1),
                                dict(hq=7), dict(hkv=0), dict(hkv=3), dict(d=32), dict(d=256), dict(page=128), dict(split=-1), dict(split=2 ** 25), dict(pages=0),
                                dict(pages=2 ** 26), dict(max_pages=-1), dict(window=-1), dict(cap=-1.0), dict(cap=float("nan")), dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=float("inf")), dict(cu=None, T=3),
                                dict(cu=None, most=2), dict(hq=2 ** 20, hkv=2 ** 20, ldq=2 ** 27, ldo=2 ** 27), dict(hq=4097, hkv=1, ldq=2 ** 20, ldo=2 ** 20), dict(work=OK + 4)])
def test_attention_refusals(kw):
    assert attn(**kw) == 1


def gemm(x=OK, ldx=256, w=OK, out=OK, ldo=64, r=None, ldr=0, bias=None, M=4, N=64, K=256, epi=0):
    return L.hbk_gemm_q4(x, ldx, w, out, ldo, r, ldr, bias, M, N, K, epi, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(out=None), dict(x=OK + 2), dict(w=OK + 4), dict(out=OK + 1), dict(out=OK + 2, epi=6), dict(ldx=248), dict(ldx=260),
                                dict(ldo=63), dict(M=-1), dict(M=257), dict(N=0), dict(K=0), dict(K=48), dict(epi=2), dict(epi=5), dict(epi=7), dict(epi=-1), dict(epi=1), dict(epi=3),
                                dict(epi=4, bias=OK), dict(epi=4, r=OK, ldr=64), dict(epi=3, r=OK, ldr=63), dict(epi=3, r=OK + 1, ldr=64), dict(epi=1, bias=OK + 1)])
def test_product_refusals(kw):
    assert gemm(**kw) == 1


@pytest.mark.parametrize("blocks,packed,N,K", [(None, OK, 16, 128), (OK, None, 16, 128), (OK, OK + 8, 16, 128), (OK, OK, 0, 128), (OK, OK, 16, 100), (OK, OK, 16, 0)])
def test_pack_refusals(blocks, packed, N, K):
    assert L.hbk_gemm_q4_pack(blocks, packed, N, K, None) == 1


def test_sizes():
    assert L.hbk_kv_q4_plane_bytes(10, 8, 128) == 10 * 8 * (64 * 64 + 64 * 4 * 2) and L.hbk_kv_q4_plane_bytes(3, 1, 64) == 3 * (64 * 32 + 64 * 2 * 2)
    assert [L.hbk_kv_q4_plane_bytes(*a) for a in ((0, 1, 64), (1, 0, 64), (1, 1, 96))] == [0, 0, 0]
    assert L.hbk_kv_q4_plane_bytes(2 ** 24, 8, 128) == 2 ** 27 * 4608
    assert L.hbk_gemm_q4_bytes(16, 128) == 1152 and L.hbk_gemm_q4_bytes(17, 160) == 4 * 1152 and L.hbk_gemm_q4_bytes(28672, 4096) == 28672 * 4096 * 9 // 16
    assert [L.hbk_gemm_q4_bytes(*a) for a in ((0, 128), (16, 0), (16, 48))] == [0, 0, 0]


@pytest.mark.parametrize("B,most,longest,hq,hkv,window", [(1, 1, 777, 32, 8, 0), (32, 1, 2176, 32, 8, 0), (3, 1, 131000, 32, 8, 0), (1, 1, 1, 1, 1, 0), (96, 1, 6000, 32, 8, 4096),
                                                         (3, 97, 5000, 12, 2, 0), (1, 300, 70000, 9, 3, 100), (65535, 1, 100, 8, 8, 0), (1, 1, 0, 8, 8, 0)])
def test_shares_cover_what_is_seen_and_fit_the_workspace(B, most, longest, hq, hkv, window):
    split = L.hbk_attn_paged_q4_split(B, most, longest, hq, hkv, window, 148)
    group = hq // hkv
    cols = 16 if group * most > 8 else 8
    assert 4 <= split <= 40
    n = L.hbk_attn_paged_q4_workspace_floats(B, B * most, most, longest, hq, hkv, 128, split, window)
    shares = n // (B * most * hq * 132) if n else 1
    assert n == (0 if shares == 1 else B * most * hq * 132 * shares)
    for length in {longest, longest - 1, longest // 2, 65 % (longest + 1), min(longest, split * 64 + 1)}:
        for c0 in range(0, group * most, cols):
            first, last = c0 // group, (min(c0 + cols, group * most) - 1) // group
            hi = max(length - most + last + 1, 0)
            lo = max(length - most + first - window + 1, 0) if window else 0
            if hi > lo:
                assert -(-(-(-hi // 64) - lo // 64) // split) <= shares


def test_split_refusals():
    assert [L.hbk_attn_paged_q4_split(*a) for a in ((0, 1, 10, 8, 8, 0, 148), (1, 0, 10, 8, 8, 0, 148), (1, 1, -1, 8, 8, 0, 148), (1, 1, 10, 8, 3, 0, 148), (1, 1, 10, 8, 8, -1, 148),
                                                            (1, 1, 10, 8, 8, 0, -1))] == [-1] * 6
    assert L.hbk_attn_paged_q4_workspace_floats(1, 1, 1, 10, 8, 3, 128, 1, 0) == 0


def test_the_limit_of_waits():
    former = L.hbk_attn_paged_q4_wait_cycles(7)
    assert former > 10 ** 9 and L.hbk_attn_paged_q4_wait_cycles(former) == 7


@pytest.mark.parametrize("B,rows,longest,hq,hkv,d,window", [(1, 8192, 131072, 32, 8, 128, 0), (1, 131072, 131072, 32, 8, 128, 0), (1, 131072, 131072, 64, 8, 64, 0), (4, 32768, 131072, 32, 8, 128, 0),
                                                            (64, 63, 131072, 32, 8, 128, 0), (1, 50000, 2 ** 20, 16, 1, 128, 0), (512, 8, 131072, 32, 8, 128, 0), (1, 65536, 131072, 32, 8, 128, 9000),
                                                            (1024, 1, 131072, 128, 8, 128, 0)])
def test_the_rule_bounds_the_workspace(B, rows, longest, hq, hkv, d, window):
    """By the rule a call of many rows has shares as long as keep the workspace within a GiB, and none where two to a column would already take more."""
    split = L.hbk_attn_paged_q4_split(B, rows, longest, hq, hkv, window, 148)
    n = L.hbk_attn_paged_q4_workspace_floats(B, B * rows, rows, longest, hq, hkv, d, split, window)
    assert split >= 4 and 0 <= n <= 2 ** 28
    column = B * rows * hq * 132
    if n == 0:
        assert 2 * column > 2 ** 28


@pytest.mark.parametrize("B,rows,longest,hq,hkv,window,split", [(1, 512, 4096, 32, 8, 0, 32), (3, 97, 5000, 12, 2, 0, 9), (1, 2048, 2048, 32, 8, 0, 32), (1, 2048, 65536, 32, 8, 0, 64),
                                                               (16, 64, 131072, 32, 8, 0, 64), (3, 1, 131000, 32, 8, 0, 32), (32, 1, 2176, 32, 8, 0, 34)])
def test_the_rule_elsewhere_is_as_it_was(B, rows, longest, hq, hkv, window, split):
    assert L.hbk_attn_paged_q4_split(B, rows, longest, hq, hkv, window, 148) == split


def test_sizes_that_the_call_refuses_have_no_split_and_no_workspace():
    assert attn(hq=65536, hkv=65536, ldq=2 ** 23, ldo=2 ** 23) == 1
    for hq, rows in ((65536, 1), (65535, 2 ** 15)):
        assert L.hbk_attn_paged_q4_split(1, rows, 1000, hq, hq, 0, 148) == -1 and L.hbk_attn_paged_q4_workspace_floats(1, 1, rows, 1000, hq, hq, 64, 4, 0) == 0
    assert L.hbk_attn_paged_q4_split(1, 131072, 131072, 64, 8, 0, 148) == 2048 and L.hbk_attn_paged_q4_split(1, 1, 1000, 65535, 65535, 0, 148) > 0


@pytest.mark.parametrize("B,most,longest,hq,hkv,window", [(3, 97, 5000, 12, 2, 0), (1, 300, 70000, 9, 3, 100), (1, 300, 70000, 9, 3, 20), (1, 2048, 2048, 32, 8, 0), (2, 512, 40000, 32, 8, 1),
                                                         (1, 40, 9000, 56, 7, 4033), (1, 700, 3000, 5, 5, 64), (4, 100, 70000, 40, 1, 63), (1, 1, 3000, 300, 1, 65), (1, 256, 5000, 1, 1, 1000),
                                                         (1, 8192, 131072, 32, 8, 0), (1, 8192, 131072, 32, 8, 30000), (2, 3, 20000, 4096, 1, 129), (5, 60, 3000, 12, 4, 127), (1, 20, 4000, 12, 1, 62)])
def test_shares_of_wide_tiles_fit_the_workspace(B, most, longest, hq, hkv, window):
    """Tiles of 128 columns from 256 columns on, of 16 or 8 below: no tile of any sequence has more shares than its columns have room for, by the rule and with splits of one's
    own; windows that end on, before and behind a page's edge."""
    group = hq // hkv
    cols = 128 if group * most >= 256 else 16 if group * most > 8 else 8
    rule = L.hbk_attn_paged_q4_split(B, most, longest, hq, hkv, window, 148)
    for split in (rule, 1, 2, 3, 7):
        n = L.hbk_attn_paged_q4_workspace_floats(B, B * most, most, longest, hq, hkv, 128, split, window)
        column = B * most * hq * 132
        assert n % column == 0
        shares = max(n // column, 1)
        worst = 0
        for rows in {most, most // 2 + 1, 1}:
            for length in {longest - i for i in (0, 1, 2, 31, 32, 63, 64, 65)} | {longest // 2, most, most + window, min(longest, split * 64 + 1)}:
                if not 0 < length <= longest:
                    continue
                tiles = range(0, group * rows, cols)
                for c0 in (list(tiles) if len(tiles) < 80 else list(tiles[:40]) + list(tiles[-40:])):
                    first, last = c0 // group, (min(c0 + cols, group * rows) - 1) // group
                    hi = min(max(length - rows + last + 1, 0), length)
                    lo = max(length - rows + first - window + 1, 0) if window else 0
                    if hi > lo:
                        worst = max(worst, -(-(-(-hi // 64) - lo // 64) // split))
        assert 0 < worst <= shares and shares <= worst + 1, (split, worst, shares)  # (nor does it have room for many that are none)
