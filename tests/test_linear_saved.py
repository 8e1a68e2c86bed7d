"""The fused products' backward takes its saved tensors as they come back: hooks on saved tensors
(torch.autograd.graph.save_on_cpu) return copies that lie otherwise than what was saved."""
import contextlib

import pytest
import torch

import linear_ref as ref
from gsr_amd import _lib
from gsr_amd.linear import _Gated, _Linear, fused_linear, gated_linear

gpu = pytest.mark.gpu

LAYOUTS = {"slice": lambda v: torch.nn.functional.pad(v, (3, 3, 1, 1))[1:-1, 3:-3],
           "transposed": lambda v: v.t().contiguous().t(),
           "contiguous": lambda v: v.contiguous()}


class _Recorder:
    """libgsr's entries that note their arguments and do nothing."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def entry(*args):
            self.calls[name] = args
            return 0
        return entry


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("pair", [False, True])
def test_backward_passes_the_strides_of_what_was_unpacked(monkeypatch, layout, pair):
    """The strides given with a pointer are those of the tensor that the pointer belongs to: with
    those of the tensor that was saved, a compact copy would be read past its end."""
    lib = _Recorder()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "raw_stream", lambda dev: 0)
    d = ref.inputs(1, 6, 5, 4, torch.float32, "cpu", gated_pair=True)
    lay = LAYOUTS[layout]
    x, w0, w1 = (lay(d[n]).detach().requires_grad_(True) for n in ("x", "w0", "w1"))
    unpacked = {}

    def unpack(t):
        unpacked[t.data_ptr()] = t
        return t

    with torch.autograd.graph.saved_tensors_hooks(
            lambda t: t.clone(memory_format=torch.contiguous_format), unpack):
        y = _Gated.apply(x, w0, w1, d["b0"], d["b1"], 3) if pair else _Linear.apply(x, w0, d["b0"], None, 3)
        torch.autograd.grad(y, (x, w0), torch.ones_like(y))
    args = lib.calls["gsr_gated_backward" if pair else "gsr_linear_backward"]
    if pair:
        given = [(args[4], args[5], 1), (args[6], args[8], 1), (args[7], args[8], 1)]
    else:
        given = [(args[4], args[5], args[6]), (args[7], args[8], 1)]
    for pointer, row, col in given:
        assert (row, col) == unpacked[pointer].stride()


@gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("pair", [False, True])
def test_gradients_with_saved_tensors_on_the_host(layout, pair, t):
    """Activations kept in host memory between the passes give the gradients of those that stayed."""
    d = ref.inputs(2, 90, 37, 53, t, "cuda", gated_pair=pair)
    for n in ("x", "w0", "w1"):
        if n in d:
            d[n] = LAYOUTS[layout](d[n])
    names = [n for n in ("x", "w0", "w1", "b0", "b1") if n in d]
    results = []
    for context in (contextlib.nullcontext(), torch.autograd.graph.save_on_cpu()):
        v = {n: d[n].detach().requires_grad_(True) for n in names}
        with context:
            y = (gated_linear(v["x"], v["w0"], v["w1"], v["b0"], v["b1"], activation="gelu") if pair
                 else fused_linear(v["x"], v["w0"], v["b0"], activation="gelu"))
        results.append(torch.autograd.grad(y, [v[n] for n in names], d["dy"]))
    for n, a, b in zip(names, *results):
        assert torch.equal(a, b), n
