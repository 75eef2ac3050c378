"""The calls of 8-bit products and of token scores that are refused, and their host arithmetic (no GPU: nothing is launched)."""
import pytest

import helix_b200 as hb

L = hb.load_library()
OK = 4096  # an address that is aligned; refused calls never look at it


def rows(x=OK, f32=0, ldx=256, codes=OK, ldc=256, scales=OK, seen=None, lds=0, T=3, K=256):
    return L.hbk_rows_q8(x, f32, ldx, codes, ldc, scales, seen, lds, T, K, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(codes=None), dict(scales=None), dict(x=OK + 8), dict(codes=OK + 8), dict(scales=OK + 2), dict(ldx=248), dict(ldx=260), dict(ldc=248), dict(ldc=264),
                                dict(f32=1, ldx=252), dict(f32=1, x=OK + 4), dict(f32=1, ldx=260), dict(seen=OK, lds=248), dict(seen=OK, lds=260), dict(seen=OK + 2, lds=256), dict(T=-1), dict(K=0),
                                dict(K=-1), dict(K=2 ** 30 + 1, ldx=2 ** 31 - 8, ldc=2 ** 31 - 16), dict(T=2 ** 30 + 1)])
def test_rows_refusals(kw):
    assert rows(**kw) == 1 and b"invalid argument" in L.hbk_last_error()


def gemm(x=OK, ldx=256, xs=OK, w=OK, ldw=256, ws=OK, out=OK, ldo=64, r=None, ldr=0, bias=None, M=4, N=64, K=256, epi=0):
    return L.hbk_gemm_q8(x, ldx, xs, w, ldw, ws, out, ldo, r, ldr, bias, M, N, K, epi, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None), dict(x=OK + 8), dict(xs=OK + 2), dict(w=OK + 8), dict(ws=OK + 4), dict(out=OK + 8), dict(ldx=240),
                                dict(ldx=264), dict(ldw=240), dict(ldw=264), dict(ldo=56), dict(ldo=68), dict(ldo=66, epi=6), dict(M=-1), dict(N=0), dict(K=0), dict(K=131057, ldx=131072, ldw=131072),
                                dict(epi=-1), dict(epi=7), dict(epi=8), dict(epi=1), dict(epi=2), dict(epi=3), dict(epi=4, bias=OK), dict(epi=4, r=OK, ldr=64), dict(epi=3, r=OK, ldr=56),
                                dict(epi=3, r=OK, ldr=68), dict(epi=3, r=OK + 8, ldr=64), dict(epi=1, bias=OK + 2), dict(epi=5), dict(epi=5, N=320), dict(epi=5, N=256, ldo=120), dict(M=2 ** 30 + 1), dict(N=2 ** 30 + 1, ldo=2 ** 31 - 8)])
def test_product_refusals(kw):
    assert gemm(**kw) == 1


def head(x=OK, ldx=256, xs=None, w=OK, ldw=256, ws=None, targets=OK, lp=OK, entropy=OK, work=OK, T=4, V=100, H=256, scale=1.0, cap=0.0):
    return L.hbk_head_scores(x, ldx, xs, w, ldw, ws, targets, lp, entropy, work, T, V, H, scale, cap, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(work=None), dict(targets=None), dict(lp=None, entropy=None), dict(xs=OK), dict(ws=OK), dict(x=OK + 8), dict(w=OK + 2), dict(ldx=248),
                                dict(ldx=260), dict(ldw=248), dict(ldw=260), dict(xs=OK, ws=OK, ldx=264), dict(xs=OK, ws=OK + 4), dict(xs=OK + 1, ws=OK), dict(work=OK + 2), dict(targets=OK + 2),
                                dict(lp=OK + 1), dict(entropy=OK + 2), dict(T=-1), dict(T=2 ** 28 + 1), dict(V=0), dict(V=2 ** 30 + 1), dict(H=0), dict(xs=OK, ws=OK, H=131057, ldx=131072, ldw=131072),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf"))])
def test_head_refusals(kw):
    assert head(**kw) == 1


def scores(x=OK, f32=1, ldl=104, targets=OK, T=4, V=100, top=3, lp=OK, rank=OK, entropy=OK, ids=OK, top_lp=OK):
    return L.hbk_token_scores(x, f32, ldl, targets, T, V, top, lp, rank, entropy, ids, top_lp, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=OK + 8), dict(ldl=96), dict(ldl=108), dict(f32=0, ldl=100), dict(targets=None), dict(targets=None, lp=None), dict(targets=None, rank=None), dict(ids=None),
                                dict(targets=OK + 2), dict(lp=OK + 2), dict(rank=OK + 1), dict(entropy=OK + 2), dict(ids=OK + 2), dict(top_lp=OK + 1), dict(T=-1), dict(T=2 ** 28 + 1), dict(V=0),
                                dict(V=2 ** 30 + 1, ldl=2 ** 30 + 8), dict(top=-1), dict(top=65), dict(top=5, V=4)])
def test_token_scores_refusals(kw):
    assert scores(**kw) == 1


def test_nothing_to_do_is_no_error():
    assert rows(T=0) == 0 and gemm(M=0) == 0 and head(T=0) == 0 and scores(T=0) == 0


def test_workspace():
    assert L.hbk_head_scores_workspace_floats(0, 5) == 0 and L.hbk_head_scores_workspace_floats(4, 0) == 0 and L.hbk_head_scores_workspace_floats(-1, 4) == 0
    for T, V in ((1, 1), (32, 128256), (128, 129), (129, 257), (2048, 128256), (100000, 151936)):
        n = L.hbk_head_scores_workspace_floats(T, V)
        tiles = -(-V // (128 if T <= 128 else 256))
        assert n == T * (12 * tiles + 1)


def test_the_limit_of_waits():
    former = L.hbk_q8_wait_cycles(7)
    assert former > 10 ** 9 and L.hbk_q8_wait_cycles(former) == 7
