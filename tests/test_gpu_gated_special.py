"""NaN and infinities in the block operators' inputs, through each of their kernels: they stay where the formulas put them, and
every other value keeps its bits. And the large kernels captured into graphs, and calls of two threads at once."""
import threading

import pytest
import torch

import gated_ref as ref
from test_gpu_gated import BF, F16, F32, code, k, rnd  # noqa: F401 (k: the fixture)

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")

# few rows with 8 and 16 features a workgroup, with 32 (8-bit save); 64 x 64, 128 x 128 tiles; two workgroups to a CU; D is no
# multiple of a K-step, and rows and features end inside a tile
FORWARD = [(5, 72, 40), (40, 72, 40), (16, 72, 2056), (70, 72, 48), (520, 136, 3000), (25601, 72, 136)]


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def pattern(got, want):
    """NaN and infinities of got are those of want."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())


@pytest.mark.parametrize("M,D,F", FORWARD)
@pytest.mark.parametrize("dtype,act,save", [(BF, "silu", "16"), (F16, "gelu", "8"), (BF, "relu", "8"), (F16, "none", "16"), (BF, "gelu", None)])
def test_gated_forward(k, M, D, F, dtype, act, save):  # noqa: F811
    x, w, b = rnd(1, M, D, dtype=dtype), rnd(2, 2 * F, D, scale=0.2, dtype=dtype), 0.1 * rnd(3, 2 * F)

    def run(x, w, b):
        out = torch.empty(M, F, device="cuda", dtype=dtype)
        kept = {"8": lambda: k.q8_empty((M, 2, F), "cuda"), "16": lambda: torch.empty(M, 2 * F, device="cuda", dtype=dtype)}.get(save, lambda: None)()
        k.gated_fwd(x, w, out, act=code(act), bias=b, save=kept)
        return out, k.dequant8(*kept, torch.empty(M, 2, F, device="cuda")).view(M, 2 * F) if save == "8" else kept
    clean, kept0 = run(x, w, b)
    rows, feats = [M // 2, M - 1], [F // 3, F - 1]
    x2, w2, b2 = x.clone(), w.clone(), b.clone()
    x2[rows[0], D - 1], x2[rows[1], 0] = NAN, INF
    w2[feats[0], 3], b2[F + feats[1]] = NAN, -INF
    out, kept = run(x2, w2, b2)
    gu, h = ref.gated_fwd(x2, w2, act, b2)
    pattern(out[rows], h[rows])
    pattern(out[:, feats], h[:, feats])
    r = torch.ones(M, dtype=torch.bool, device="cuda")
    f = torch.ones(F, dtype=torch.bool, device="cuda")
    r[rows], f[feats] = False, False
    assert same(out[r][:, f], clean[r][:, f])
    if save == "16":
        pattern(kept, gu)
    if save == "8":
        assert torch.equal(kept.isnan(), ~gu.isfinite())
    if save:  # (an 8-bit group's other values keep theirs, but for a scale that the group's largest value took along)
        f2 = torch.cat([f, f])
        for i in feats:
            for at in (i, F + i):
                lo, half = at % F // 32 * 32, at // F * F
                f2[half + lo:half + min(lo + 32, F)] = False
        assert same(kept[r][:, f2], kept0[r][:, f2])


# 64 x 64, 128 x 128 tiles; 256 x 256 with K cut over idle workgroups
@pytest.mark.parametrize("M,D,F", [(3, 72, 40), (333, 72, 200), (1100, 520, 1032), (16400, 520, 1032)])
@pytest.mark.parametrize("dtype,act,eight", [(BF, "silu", False), (F16, "gelu", True), (BF, "gelu", False), (F16, "none", True)])
def test_gated_backward(k, M, D, F, dtype, act, eight):  # noqa: F811
    x, w = rnd(1, M, D, dtype=dtype), rnd(2, 2 * F, D, scale=D ** -0.5, dtype=dtype)
    dh, gu = rnd(3, M, F, dtype=dtype), rnd(4, M, 2 * F, dtype=dtype)

    def run(dh, gu):
        saved = tuple(t.view(M, 2, t.shape[1]) for t in k.quant8(gu.view(2 * M, F))) if eight else gu
        got = {"dx": torch.empty_like(x), "dw": torch.empty_like(w), "db": torch.empty(2 * F, device="cuda"), "h": torch.empty_like(dh)}
        k.gated_bwd(dh, saved, k.quant8(x) if eight else x, w, act=code(act), **got)
        return got
    clean = run(dh, gu)
    dh2, gu2 = dh.clone(), gu.clone()
    fa, fb = F // 2, F - 1
    dh2[M - 1, fa] = NAN
    gu2[M // 2, fb], gu2[M // 2, F + fb] = NAN, NAN  # (an infinity would be NaN in the 8-bit form)
    got = run(dh2, gu2)
    r = torch.ones(M, dtype=torch.bool, device="cuda")
    f = torch.ones(F, dtype=torch.bool, device="cuda")
    r[[M - 1, M // 2]] = False
    f[[fa, fb]] = False
    assert bool(got["dx"][~r].isnan().all()) and same(got["dx"][r], clean["dx"][r])
    f2 = torch.cat([f, f])
    assert bool(got["dw"][~f2].isnan().all()) and same(got["dw"][f2], clean["dw"][f2])
    assert bool(got["db"][~f2].isnan().all()) and same(got["db"][f2], clean["db"][f2])
    assert bool(got["h"][M // 2, fb].isnan()) and same(got["h"][r], clean["h"][r])
    if not eight:  # infinite gates: NaN or infinite where the formula says so
        gu2 = gu.clone()
        gu2[M - 1, fa], gu2[M // 2, fb] = INF, -INF
        got, want = run(dh, gu2), ref.gated_bwd(dh, gu2, x, w, act)
        pattern(got["h"], want["h"])
        pattern(got["db"], want["db"])
        assert same(got["dw"][f2], clean["dw"][f2]) and same(got["dx"][r], clean["dx"][r])


@pytest.mark.parametrize("rows,d", [(33, 96), (33, 250), (33, 256), (33, 1000), (33, 1021), (5, 2000), (5, 3000), (5, 4001), (5, 8200), (700, 96)])
@pytest.mark.parametrize("dtype,eight", [(BF, False), (F32, False), (F16, True)])
def test_norm_backward(k, rows, d, dtype, eight):  # noqa: F811
    w, s, dy, dres = 1 + 0.2 * rnd(1, d), rnd(2, rows, d), rnd(3, rows, d, dtype=dtype), rnd(4, rows, d, dtype=dtype)
    rstd = torch.rsqrt(s.square().mean(-1) + 1e-6)

    def run(s, dy, dres):
        return k.rmsnorm_bwd(dy, k.quant8(s) if eight else s.to(dtype), rstd, w, torch.empty_like(dy), dres=dres)
    dx0, dw0 = run(s, dy, dres)
    s2, dy2, dres2 = s.clone(), dy.clone(), dres.clone()
    s2[rows - 1, d - 1], dy2[rows // 2, d // 2], dres2[0, 0], dres2[0, 1] = NAN, INF, INF, NAN
    dx, dw = run(s2, dy2, dres2)
    r, c = torch.ones(rows, dtype=torch.bool, device="cuda"), torch.ones(d, dtype=torch.bool, device="cuda")
    r[[rows - 1, rows // 2]], c[[d - 1, d // 2]] = False, False
    assert bool(dx[rows - 1].isnan().all()) and not bool(dx[rows // 2].isfinite().any())
    assert bool(dx[0, 0].isposinf()) and bool(dx[0, 1].isnan())
    dx[0, :2] = dx0[0, :2]
    assert same(dx[r], dx0[r]) and same(dw[c], dw0[c])
    assert bool(dw[d - 1].isnan()) and bool(dw[d // 2].isinf())


@pytest.mark.parametrize("M,D,F,eight", [(16400, 520, 1032, False), (4096, 768, 2048, True)])
def test_large_kernels_in_graphs(k, M, D, F, eight):  # noqa: F811
    """Forward and backward of the large tiles, captured and replayed on new inputs between eager calls."""
    def inputs(seed):
        return rnd(seed, M, D, dtype=BF), rnd(seed + 1, 2 * F, D, scale=D ** -0.5, dtype=BF), rnd(seed + 2, M, F, dtype=BF)

    def run(x, w, dh):
        h = torch.empty(M, F, device="cuda", dtype=BF)
        kept = k.q8_empty((M, 2, F), "cuda") if eight else torch.empty(M, 2 * F, device="cuda", dtype=BF)
        k.gated_fwd(x, w, h, save=kept)
        got = {"dx": torch.empty_like(x), "dw": torch.empty_like(w), "db": torch.empty(2 * F, device="cuda")}
        k.gated_bwd(dh, kept, k.quant8(x) if eight else x, w, **got)
        return dict(got, h=h)
    fixed = inputs(1)
    run(*fixed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*fixed)
    for seed in (1, 10, 20):
        new = inputs(seed)
        for a, b in zip(fixed, new):
            a.copy_(b)
        graph.replay()
        want = run(*new)
        torch.cuda.synchronize()
        for name in want:
            assert same(out[name], want[name]), (seed, name)


def test_two_threads(k):  # noqa: F811
    """Calls of two threads, each on a stream of its own and of sizes of its own, give what they give alone."""
    def work(M, D, F, seed):
        x, w = rnd(seed, M, D, dtype=BF), rnd(seed + 1, 2 * F, D, scale=D ** -0.5, dtype=BF)
        dh, gu = rnd(seed + 2, M, F, dtype=BF), rnd(seed + 3, M, 2 * F, dtype=BF)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        k.gated_bwd(dh, gu, x, w, dx=dx, dw=dw)
        return dx, dw
    jobs = [(300, 264, 200, 1), (1100, 520, 1032, 50)]
    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    got = [None, None]

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = work(*jobs[i])
            torch.cuda.current_stream().synchronize()
    ts = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    for a, b in zip(got, want):
        assert same(a[0], b[0]) and same(a[1], b[1])


@pytest.mark.parametrize("rows,d", [(33, 96), (33, 250), (17, 1000), (9, 3000), (9, 4001), (9, 8200)])
@pytest.mark.parametrize("xt,rt", [(BF, BF), (F16, F32), (F32, F32)])
def test_norm_forward_in_place(k, rows, d, xt, rt):  # noqa: F811
    """The sum over the residual and the output over x in one call; the sum over x; all with the 8-bit form beside them."""
    x, r, w = rnd(1, rows, d, dtype=xt), rnd(2, rows, d, dtype=rt), 1 + 0.2 * rnd(3, d)

    def run(x, r, y, s):
        q, rstd = k.q8_empty((rows, d), "cuda"), torch.empty(rows, device="cuda")
        k.rmsnorm_fwd(x, w, 1e-6, y, residual=r, sum_out=s, q8=q, rstd=rstd)
        return y, s, q[0], q[1], rstd
    want = run(x, r, torch.empty_like(x), torch.empty_like(r))
    x2, r2 = x.clone(), r.clone()
    for a, b in zip(run(x2, r2, x2, r2), want):
        assert same(a, b)
    if xt == rt:
        x2 = x.clone()
        for a, b in zip(run(x2, r, torch.empty_like(x), x2), want):
            assert same(a, b)
