"""The scratch sizes of every entry at the ends of the ranges that the header allows: a number for
each, on the host, where a division by no rows would end the process."""
import pytest

from gsr_amd import _lib


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("K,N", [(1, 1), (12, 20), (1, 4096), (4096, 1), (600, 600), (4096, 4096), (1 << 22, 1 << 21)])
def test_no_rows(kind, K, N):
    L = _lib.load()
    assert L.gsr_linear_scratch_bytes(kind, 0, K, N) >= 0 and L.gsr_gated_scratch_bytes(kind, 0, K, N) >= 0
    for need in (0, 1, 2):
        # no rows: no gradients to keep and none to sum
        assert L.gsr_gated_backward_scratch_bytes(kind, 0, K, N, need) <= 256
        for act in range(4):
            assert L.gsr_linear_backward_scratch_bytes(kind, 0, K, N, act, need) <= 256


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("M", [1, 63, 64, 65, 255, 256, 257, 8191, 8192, 8193, 32767, 32768, 1 << 20, 1 << 36])
@pytest.mark.parametrize("K,N", [(1, 1), (1, 4096), (4096, 1), (257, 513), (4100, 130), (4096, 4096)])
def test_rows(kind, M, K, N):
    """A backward with weight gradients needs no less than one without, and each a sum of at least
    its own gradients before the activation."""
    L = _lib.load()
    size = 4 if kind == 0 else 2
    assert L.gsr_linear_scratch_bytes(kind, M, K, N) >= 0 and L.gsr_gated_scratch_bytes(kind, M, K, N) >= 0
    for act in range(4):
        a, b, c = (L.gsr_linear_backward_scratch_bytes(kind, M, K, N, act, need) for need in (0, 2, 1))
        assert (M * N * size if act else 0) <= a <= b <= c
    a, b, c = (L.gsr_gated_backward_scratch_bytes(kind, M, K, N, need) for need in (0, 2, 1))
    assert 2 * M * N * size <= a <= b <= c


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("pair", [False, True])
def test_gradients_of_no_rows_and_wide_layers(kind, pair):
    import torch

    from gsr_amd.linear import fused_linear, gated_linear
    t = (torch.float32, torch.float16, torch.bfloat16)[kind]
    for K, N in ((600, 2100), (2100, 600)):
        x = torch.empty(0, K, dtype=t, device="cuda", requires_grad=True)
        w, u = (torch.ones(N, K, dtype=t, device="cuda", requires_grad=True) for _ in range(2))
        b = torch.ones(N, dtype=t, device="cuda", requires_grad=True)
        y = gated_linear(x, w, u, b) if pair else fused_linear(x, w, b, activation="gelu")
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert dx.shape == (0, K) and not bool(dw.any()) and not bool(db.any())


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_which_sums_of_few_rows_are_cut(kind):
    """Ranges of a long sum need scratch memory: few outputs of a long sum are cut, weights that stream
    past one block of rows, and short sums, are not."""
    L = _lib.load()
    for size in (L.gsr_linear_scratch_bytes, L.gsr_gated_scratch_bytes):
        for M, K, N in ((64, 4096, 512), (64, 4096, 1024), (128, 8192, 1024), (17, 8192, 1000)):
            assert size(kind, M, K, N) > 0, (M, K, N)
        for M, K, N in ((1, 4096, 8192), (16, 2048, 5504), (5, 512, 512), (64, 1024, 1024), (256, 512, 512)):
            assert size(kind, M, K, N) == 0, (M, K, N)
