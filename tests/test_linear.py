"""Fused linear layer and gated pair (gsr_amd.linear) against 64 bits: sizes, types, layouts,
activations, gradients, streams, graphs, and what they refuse."""
import pytest
import torch

import linear_ref as ref
from gsr_amd.linear import fused_linear, gated_linear

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = {torch.float32: "fp32", torch.float16: "fp16", torch.bfloat16: "bf16"}


def _linear(d, act, r=None):
    return fused_linear(d["x"], d["w0"], d.get("b0"), activation=act, residual=d.get("r"))


def _gated(d, act):
    return gated_linear(d["x"], d["w0"], d["w1"], d.get("b0"), d.get("b1"), activation=act)


def _want(d, act, grads=True):
    e = {k: v.detach().double() for k, v in d.items()}
    t = d["x"].dtype
    dy = e["dy"] if grads else None
    if "w1" in d:
        return ref.gated(e["x"], e["w0"], e["w1"], e.get("b0"), e.get("b1"), act, t, dy)
    return ref.linear(e["x"], e["w0"], e.get("b0"), e.get("r"), act, t, dy)


def _run(d, act, grads=True):
    names = [n for n in ("x", "w0", "w1", "b0", "b1", "r") if n in d] if grads else []
    for n in names:
        d[n] = d[n].detach().requires_grad_(True)
    y = _gated(d, act) if "w1" in d else _linear(d, act)
    got = {"y": y.detach()}
    if grads:
        got.update(zip(names, torch.autograd.grad(y, [d[n] for n in names], d["dy"])))
        r = got.pop("r", None)
        if r is not None:
            assert torch.equal(r, d["dy"])
    return got


# one of each: single elements, below / at / above a tile, odd widths, long sums, few rows against
# wide weights, many rows against a narrow output
SIZES = [(1, 1, 1), (1, 512, 512), (2, 3, 5), (5, 4096, 33), (17, 129, 1000), (31, 64, 64), (33, 100, 66),
         (64, 64, 64), (65, 65, 65), (127, 31, 129), (128, 128, 128), (129, 256, 257),
         (300, 7, 1), (512, 1, 16), (777, 161, 203), (2049, 96, 40), (3000, 33, 130), (4100, 31, 70), (5000, 100, 129),
         # enough rows for the kernel that keeps its rows: 1, 2, 4, 6 and 8 steps of 32 inputs
         (32769, 31, 70), (32800, 3, 64), (33000, 63, 33), (32768, 128, 64), (32771, 161, 203),
         (32900, 256, 130), (33001, 250, 40),
         # the largest tiles, operands straight to LDS, the last step of either sum ragged; the same
         # sizes where nothing is aligned; a narrow weight gradient
         (33001, 264, 264), (16500, 72, 1032), (33001, 263, 265), (20000, 40, 200),
         # around the sizes where few rows end
         (32, 520, 640), (33, 520, 640), (63, 520, 640), (66, 520, 640), (129, 520, 640),
         (256, 520, 640), (257, 520, 640),
         # few tiles and long sums
         (300, 4100, 130), (40, 700, 2101), (66, 1024, 2052), (4099, 600, 64), (8190, 2100, 33),
         (20, 130, 4097)]


@gpu
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_sizes(M, K, N, t):
    act = ("gelu", "silu", "relu", "none")[(M + K + N) % 4]
    d = ref.inputs(M * 7 + N, M, K, N, t, "cuda", bias=(M + K) % 3 != 0, residual=N % 2 == 1)
    ref.check(_run(d, act), _want(d, act), f"{M}x{K}x{N} {act}")


@gpu
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_gated_sizes(M, K, N, t):
    act = ("gelu", "silu", "relu")[(M + K + N) % 3]
    d = ref.inputs(M * 5 + N, M, K, N, t, "cuda", gated_pair=True, bias=(M + N) % 3 != 0)
    ref.check(_run(d, act), _want(d, act), f"{M}x{K}x{N} {act}")


@gpu
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_activations_far_from_zero(act, t):
    """Arguments from -60 to 60: tails, saturation, nothing but finite values."""
    d = ref.inputs(3, 200, 32, 48, t, "cuda", residual=True, spread=12.0)
    got = _run(d, act)
    assert all(bool(torch.isfinite(v).all()) for v in got.values())
    ref.check(got, _want(d, act), act)


@gpu
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("K", [1, 3, 16, 61])
@pytest.mark.parametrize("M", [1, 2, 63, 1000, 33003])
def test_channel_major_input(M, K, t):
    """A [K,H,W] image read as its transpose, in place; its gradient reaches the image."""
    d = ref.inputs(M + K, M, K, 40, t, "cuda")
    image = d["x"].t().contiguous().requires_grad_(True)
    y = fused_linear(image.t(), d["w0"], d["b0"], activation="silu")
    (g,) = torch.autograd.grad(y, image, d["dy"])
    ref.check({"y": y.detach(), "x": g.t()}, _want(d, "silu"))


@gpu
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("pair", [False, True])
def test_strides_and_alignment(t, pair):
    """Slices of larger tensors at odd offsets, transposed weights, expanded rows, a gradient that
    is a slice: the values are those of contiguous copies."""
    d = ref.inputs(11, 90, 37, 53, t, "cuda", gated_pair=pair, residual=not pair)
    plain = _run(dict(d), "gelu")

    def inside(m):  # a view with a row stride and a base that no vector divides
        big = torch.full((m.shape[0] + 2, m.shape[1] + 6), float("nan"), dtype=t, device="cuda")
        v = big[1:-1, 3:-3]
        v.copy_(m)
        return v

    for change in (lambda n, v: inside(v) if v.dim() == 2 else v,
                   lambda n, v: v.t().contiguous().t() if v.dim() == 2 else v):
        e = {n: change(n, v.detach()) for n, v in d.items()}
        assert any(not v.is_contiguous() for v in e.values())
        got = _run(e, "gelu")
        for n, v in got.items():
            ref.check({n: v}, _want(d, "gelu"), "strided")
    rows = {**d, "x": d["x"].detach()[:1].expand(90, 37)}
    ref.check(_run(dict(rows), "gelu"), _want(rows, "gelu"), "expanded")
    lead = {**{n: v.detach() for n, v in d.items()}}
    for n in ("x", "r", "dy"):
        if n in lead:
            lead[n] = lead[n].reshape(2, 5, 9, -1)
    got = _run(lead, "gelu")
    assert got["y"].shape == (2, 5, 9, 53) and got["x"].shape == (2, 5, 9, 37)
    for n in got:
        assert torch.equal(got[n].reshape(plain[n].shape), plain[n])


@gpu
def test_broadcast_gradients():
    """A residual and a row shared by expand(): autograd sums the gradient over the copies."""
    d = ref.inputs(5, 64, 20, 30, torch.float32, "cuda")
    r = torch.randn(30, device="cuda", requires_grad=True)
    y = fused_linear(d["x"], d["w0"], d["b0"], activation="relu", residual=r.expand(64, 30))
    (g,) = torch.autograd.grad(y, r, d["dy"])
    torch.testing.assert_close(g, d["dy"].sum(0), rtol=64 * 2 ** -24, atol=64 * 2 ** -22)
    # the same weight in two layers, the same tensor in two places
    w = (d["w0"][:20] @ d["w0"][:20].t()).detach().requires_grad_(True)
    x = d["x"].detach().requires_grad_(True)
    y = fused_linear(fused_linear(x, w, activation="silu", residual=x), w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    x2, w2 = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    y2 = (torch.nn.functional.silu(x2 @ w2.t()) + x2) @ w2.t()
    ex, ew = torch.autograd.grad(y2.sum(), (x2, w2))
    for got, want in ((gx, ex), (gw, ew)):
        assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())


@gpu
@pytest.mark.parametrize("pair", [False, True])
def test_gradients_against_differences(pair):
    """d(sum(c y))/dv along random directions against central differences of the 64-bit formula:
    relative 1e-4 (the step's own error is about h^2 = 1e-8 relative, the kernel's 1e-6)."""
    d = ref.inputs(9, 40, 24, 36, torch.float32, "cuda", gated_pair=pair, residual=not pair)
    got = _run(d, "silu")
    e = {n: v.detach().double() for n, v in d.items()}

    def loss(v):
        a = torch.nn.functional.silu(v["x"] @ v["w0"].t() + v["b0"])
        y = a * (v["x"] @ v["w1"].t() + v["b1"]) if pair else a + v["r"]
        return float((y * e["dy"]).sum())

    for n in got:
        if n == "y":
            continue
        way = torch.randn(e[n].shape, generator=torch.Generator().manual_seed(1)).double().cuda()
        h = 1e-4
        diff = (loss({**e, n: e[n] + h * way}) - loss({**e, n: e[n] - h * way})) / (2 * h)
        along = float((got[n].double() * way).sum())
        assert abs(along - diff) <= 1e-4 * max(1.0, abs(diff)), n


@gpu
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_no_rows(t):
    d = ref.inputs(1, 0, 12, 20, t, "cuda", residual=True)
    got = _run(d, "gelu")
    assert got["y"].shape == (0, 20) and got["x"].shape == (0, 12)
    assert not got["w0"].any() and not got["b0"].any()
    d = ref.inputs(1, 0, 12, 20, t, "cuda", gated_pair=True)
    got = _run(d, "gelu")
    assert got["y"].shape == (0, 20) and not got["w1"].any() and not got["b1"].any()


@gpu
@pytest.mark.parametrize("M", [3, 300, 33000])
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_infinities_and_nan_stay_where_they_are(t, M):
    """A row with an infinity or a NaN spoils that row as 64-bit arithmetic says, and no other."""
    d = ref.inputs(2, M, 70, 90, t, "cuda", residual=True)
    clean = _linear(d, "none")
    x = d["x"].clone()
    x[0, 5], x[1, 7], x[2, 9] = float("inf"), float("nan"), float("-inf")
    y = _linear({**d, "x": x}, "none")
    want = x.double() @ d["w0"].double().t() + d["b0"].double() + d["r"].double()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(y[:3][torch.isinf(y[:3])].double(), want[:3][torch.isinf(want[:3])])
    assert torch.equal(y[3:], clean[3:])
    # a zero weight against an infinity is a NaN
    w = d["w0"].clone()
    w[4] = 0
    assert bool(torch.isnan(_linear({**d, "x": x, "w0": w}, "none")[0, 4]))


@gpu
def test_float_range():
    """32-bit operands from 1e-30 to 1e30 whose products are of ordinary size keep 32-bit accuracy."""
    d = ref.inputs(4, 140, 50, 60, torch.float32, "cuda", bias=False)
    s = torch.logspace(-30, 30, 50, device="cuda")
    d["x"], d["w0"] = d["x"] * s, d["w0"] / s
    got = _run(d, "none")
    ref.check(got, _want(d, "none"))


@gpu
def test_rows_beyond_the_last_are_untouched():
    """The C entry writes rows [0, M) of y and columns [0, N) of a wider row, nothing else."""
    from gsr_amd import _lib
    L = _lib.load()
    for kind, t in ((0, torch.float32), (2, torch.bfloat16)):
        for M, N in ((5, 20), (130, 131), (33001, 75)):
            d = ref.inputs(6, M, 24, N, t, "cuda")
            y = torch.full((M + 3, N + 8), 7.0, dtype=t, device="cuda")
            scratch = torch.empty(L.gsr_linear_scratch_bytes(kind, M, 24, N) + 1, dtype=torch.uint8,
                                  device="cuda")
            rc = L.gsr_linear(kind, M, 24, N, d["x"].data_ptr(), 24, 1, d["w0"].data_ptr(), 24,
                              d["b0"].data_ptr(), None, 0, 1, y.data_ptr(), N + 8,
                              scratch.data_ptr(), _lib.raw_stream(y.device))
            assert rc == 0
            ref.check({"y": y[:M, :N]}, _want(d, "relu", grads=False))
            assert bool((y[M:] == 7).all()) and bool((y[:, N:] == 7).all())


@gpu
@pytest.mark.parametrize("M,K,N", [(8_400_000, 256, 256), (4_200_000, 512, 512)])
def test_more_than_2_to_31_elements(M, K, N):
    """Offsets of operands and results pass 32 bits.  Only the first and the last rows have a gradient
    that is not zero, so these rows' formulas give all gradients."""
    t, n = torch.bfloat16, 300
    d = ref.inputs(15, 2 * n, K, N, t, "cuda")
    ends = {k: d[k] for k in ("x", "dy")}
    for k, v in ends.items():
        big = torch.zeros(M, v.shape[1], dtype=t, device="cuda")
        big[:n], big[-n:] = v[:n], v[n:]
        d[k] = big
    got = _run(d, "silu")
    for k in ("y", "x"):
        got[k] = torch.cat([got[k][:n], got[k][-n:]])
    e = {**d, **ends}
    want = _want(e, "silu")
    # sums over M rows, all but 2 n of them zero: exact zeros add nothing
    ref.check(got, want)


@gpu
@pytest.mark.parametrize("pair", [False, True])
def test_same_bits_every_time_and_on_another_stream(pair):
    d = ref.inputs(8, 5000, 96, 120, torch.bfloat16, "cuda", gated_pair=pair)
    first = _run(d, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _run(d, "gelu")
    torch.cuda.current_stream().wait_stream(side)
    for n in first:
        assert torch.equal(first[n], second[n]), n


@gpu
def test_two_calls_at_once():
    """Calls on two streams, of sizes that need scratch memory, do not disturb each other."""
    sizes = [(300, 2100, 130), (33000, 64, 200)]
    ds = [ref.inputs(20 + i, *sizes[i], torch.bfloat16, "cuda") for i in range(2)]
    want = [_run(dict(d), "silu") for d in ds]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_run(dict(ds[i]), "silu"))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for n in g:
                assert torch.equal(g[n], want[i][n]), (i, n)


@gpu
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("t,M,K", [(torch.float32, 700, 40), (torch.bfloat16, 3000, 2100),
                                   (torch.float16, 33000, 40)])
def test_captured_and_replayed(pair, t, M, K):
    """Forward and backward in a graph, replayed on new values with eager calls between: each
    replay has the eager call's bits.  Two graphs of the same shapes live side by side."""
    d = ref.inputs(12, M, K, 72, t, "cuda", gated_pair=pair)
    _run(dict(d), "silu")  # builds, allocates
    torch.cuda.synchronize()
    names = [n for n in ("x", "w0", "w1", "b0", "b1") if n in d]
    graphs = []
    for _ in range(2):
        s = {n: d[n].detach().clone() for n in names + ["dy"]}
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            leaves = {n: s[n].detach().requires_grad_(True) for n in names}
            y = _gated(leaves, "silu") if pair else _linear(leaves, "silu")
            out = [y] + list(torch.autograd.grad(y, [leaves[n] for n in names], s["dy"]))
        graphs.append((g, s, out))
    for k in range(4):
        for i, (g, s, out) in enumerate(graphs):
            new = ref.inputs(100 + 2 * k + i, M, K, 72, t, "cuda", gated_pair=pair)
            for n in s:
                s[n].copy_(new[n])
            g.replay()
            eager = _run(new, "silu")
            torch.cuda.synchronize()
            for n, v in zip(["y"] + names, out):
                assert torch.equal(v, eager[n]), (k, i, n)


@gpu
def test_only_the_gradients_asked_for():
    d = ref.inputs(13, 200, 30, 50, torch.float32, "cuda", residual=True)
    full = _run(dict(d), "gelu")
    for n in ("x", "w0", "b0"):
        e = {k: v.detach() for k, v in d.items()}
        e[n].requires_grad_(True)
        y = _linear(e, "gelu")
        (g,) = torch.autograd.grad(y, e[n], d["dy"])
        assert torch.equal(g, full[n]), n
    e = ref.inputs(13, 200, 30, 50, torch.float32, "cuda", gated_pair=True)
    full = _run(dict(e), "gelu")
    for n in ("x", "w0", "w1", "b0", "b1"):
        f = {k: v.detach() for k, v in e.items()}
        f[n].requires_grad_(True)
        (g,) = torch.autograd.grad(_gated(f, "gelu"), f[n], e["dy"])
        assert torch.equal(g, full[n]), n


@gpu
def test_no_second_derivative():
    d = ref.inputs(14, 8, 8, 8, torch.float32, "cuda")
    x = d["x"].requires_grad_(True)
    (g,) = torch.autograd.grad(fused_linear(x, d["w0"], activation="silu").sum(), x,
                               create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def _cpu(M=4, K=6, N=8):
    return ref.inputs(0, M, K, N, torch.float32, "cpu", gated_pair=True, residual=True)


def test_refusals():
    d = _cpu()
    for bad, err in ((dict(activation="tanh"), ValueError), (dict(activation=None), ValueError),
                     (dict(residual=d["r"][:3]), ValueError), (dict(residual=d["r"][0]), ValueError),
                     (dict(residual=d["r"].double()), ValueError)):
        with pytest.raises(err):
            fused_linear(d["x"], d["w0"], d["b0"], **bad)
    with pytest.raises(ValueError, match="bias"):
        fused_linear(d["x"], d["w0"], d["b0"][:3])
    with pytest.raises(ValueError, match="bias"):
        fused_linear(d["x"], d["w0"], d["b0"].half())
    with pytest.raises(ValueError, match="x must have shape"):
        fused_linear(d["x"][:, :5], d["w0"])
    with pytest.raises(ValueError):
        fused_linear(d["x"], d["w0"][0])
    with pytest.raises(ValueError, match="empty"):
        fused_linear(d["x"], d["w0"][:0])
    with pytest.raises(ValueError, match="empty"):
        fused_linear(d["x"][:, :0], d["w0"][:, :0])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        fused_linear(d["x"].double(), d["w0"].double())
    with pytest.raises(TypeError):
        fused_linear(d["x"], None)
    with pytest.raises(TypeError):
        fused_linear(d["x"], d["w0"], 1.0)
    with pytest.raises(ValueError, match="up_weight"):
        gated_linear(d["x"], d["w0"], d["w1"][:7])
    with pytest.raises(ValueError, match="up_bias"):
        gated_linear(d["x"], d["w0"], d["w1"], None, d["b1"][:2])
    for call in (lambda: fused_linear(d["x"], d["w0"]), lambda: gated_linear(d["x"], d["w0"], d["w1"])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_c_entries_refuse():
    """Invalid arguments are status 1 before any GPU work (no device is touched)."""
    from gsr_amd import _lib
    L = _lib.load()
    p = 4096  # never read

    def lin(dtype=0, M=4, K=6, N=8, x=p, xr=6, xc=1, w=p, wr=6, act=0, y=p, yr=8, r=None, rr=0, s=p):
        return L.gsr_linear(dtype, M, K, N, x, xr, xc, w, wr, None, r, rr, act, y, yr, s, None)

    assert lin(dtype=3) == lin(dtype=-1) == lin(act=4) == lin(act=-1) == 1
    assert lin(M=-1) == lin(K=0) == lin(N=0) == lin(K=1 << 40) == 1
    assert lin(x=None) == lin(w=None) == lin(y=None) == 1
    assert lin(M=40000, N=80, yr=80, s=None) == 1  # this one needs scratch
    assert L.gsr_linear_scratch_bytes(0, 40000, 6, 80) > 0 == L.gsr_linear_scratch_bytes(0, 4, 6, 8)
    assert lin(xr=5) == lin(xc=2) == lin(wr=5) == lin(yr=7) == lin(r=p, rr=7) == 1
    assert lin(xr=1, xc=3) == 1
    assert lin(M=0, x=None, y=None) == 0
    assert L.gsr_linear_backward(0, 4, 6, 8, p, 6, 1, p, 6, None, 0, None, 8, p, p, p, p, None) == 1
    assert L.gsr_linear_backward(0, 4, 6, 8, p, 6, 1, p, 6, None, 0, p, 7, p, p, p, p, None) == 1
    assert L.gsr_linear_backward(0, 4, 6, 8, p, 6, 1, p, 6, None, 0, p, 8, p, p, p, None, None) == 1
    assert L.gsr_gated(0, 4, 6, 8, p, 6, p, None, 6, None, None, 3, p, 8, p, None) == 1
    assert L.gsr_gated(0, 4, 6, 8, p, 5, p, p, 6, None, None, 3, p, 8, p, None) == 1
    assert L.gsr_gated_backward(0, 4, 6, 8, p, 6, p, p, 6, None, None, 3, None, 8, p, p, p, p, None) == 1
    assert L.gsr_gated(0, 40000, 6, 80, p, 6, p, p, 6, None, None, 3, p, 80, None, None) == 1
    assert L.gsr_linear_scratch_bytes(0, -1, 6, 8) == L.gsr_gated_scratch_bytes(3, 4, 6, 8) == 0
    assert L.gsr_linear_backward_scratch_bytes(9, 4, 6, 8, 1, 1) == 0
    assert L.gsr_gated_backward_scratch_bytes(0, -4, 6, 8, 1) == 0
