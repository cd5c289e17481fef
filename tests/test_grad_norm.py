"""Global gradient norm and clip over many tensors against 64-bit sums.

The squares are summed in 64 bits, so the norm is off by the roundings of its square root's result alone: less than 2 u (u = 2^-24).  The factor
max_norm / (norm + 1e-6) adds three, its product with an element one, and a 16-bit element is rounded to its type: half a step."""
import math

import pytest
import torch

from codebase_amd import hip as h

U = 2.0**-24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def tensors(sizes, seed=0, types=TYPES, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=gen) * scale).to(types[i % len(types)]).cuda() for i, n in enumerate(sizes)]


def reference(ts, max_norm):
    norm = math.sqrt(sum(float((t.double()**2).sum()) for t in ts))
    return norm, [t.double() * min(max_norm / (norm + 1e-6), 1.0) for t in ts]


def check_clipped(got, want):
    for i, (g, w) in enumerate(zip(got, want)):
        bound = (8 * U + HALF[g.dtype] * (1 + 8 * U)) * w.abs() + TINY[g.dtype]
        assert bool(((g.double() - w).abs() <= bound).all()), i


CASES = [[1], [0, 1, 0], [3, 5], [64] * 12, [4096], [4097, 1], [100000], [1 << 20, 7, 4095, 4096, 4097], [17] * 161, [1 + 37 * i % 500 for i in range(700)],
         [3_000_001, 2_000_003]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", CASES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
def test_norm_and_clip(sizes, max_norm):
    ts = tensors(sizes)
    norm, want = reference(ts, max_norm)
    got = h.grad_norm(ts)
    assert abs(got.item() - norm) <= 2 * U * norm
    before = [t.clone() for t in ts]
    out = [torch.full_like(t, 7.0) for t in ts]
    n1 = h.clip_grad_norm(ts, max_norm, out=out)
    assert all(torch.equal(a, b) for a, b in zip(ts, before)) and torch.equal(n1, got)
    check_clipped(out, want)
    n2 = h.clip_grad_norm(ts, max_norm)
    assert torch.equal(n1, n2) and all(torch.equal(a, b) for a, b in zip(ts, out))
    if max_norm > norm:
        assert all(torch.equal(a, b) for a, b in zip(ts, before))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_unaligned_views_and_shapes(dtype):
    flat = tensors([5000], types=[dtype])[0]
    ts = [flat[1:1000].view(27, 37), flat[1000:1003], flat[1003:4999]]
    out_flat = torch.zeros(6000, dtype=dtype, device="cuda")
    outs = [out_flat[3:1002].view(27, 37), out_flat[1100:1103], out_flat[1501:5497]]
    norm, want = reference(ts, 1.0)
    got = h.clip_grad_norm(ts, 1.0, out=outs)
    assert abs(got.item() - norm) <= 2 * U * norm
    check_clipped(outs, want)
    rest = torch.ones(6000, dtype=torch.bool, device="cuda")
    for a, b in ((3, 1002), (1100, 1103), (1501, 5497)):
        rest[a:b] = False
    assert not out_flat[rest].any()


@pytest.mark.gpu
def test_tensors_without_elements():
    ts = [torch.zeros(0, device="cuda"), torch.zeros(3, 0, dtype=torch.bfloat16, device="cuda")]
    assert h.grad_norm(ts).item() == 0.0 and h.clip_grad_norm(ts, 1.0).item() == 0.0


@pytest.mark.gpu
def test_large_and_small_values():
    ts = [torch.full((1000,), 3e30, device="cuda"), torch.full((10,), 1e-30, device="cuda")]
    assert abs(h.grad_norm(ts).item() / (3e30 * math.sqrt(1000)) - 1) <= 2 * U  # the squares pass an f32's range
    small = [torch.full((4,), 1e-30, device="cuda")]
    assert abs(h.grad_norm(small).item() / 2e-30 - 1) <= 2 * U


@pytest.mark.gpu
def test_norms_that_are_not_finite():
    ts = tensors([100, 50])
    ts[0][3] = float("inf")
    n = h.clip_grad_norm(ts, 1.0)
    assert math.isinf(n.item()) and torch.isnan(ts[0][3]) and not ts[1].any() and not ts[0][4:].any()
    ts = tensors([100, 50])
    ts[1][7] = float("nan")
    n = h.clip_grad_norm(ts, 1.0)
    assert math.isnan(n.item()) and all(torch.isnan(t).all() for t in ts)


@pytest.mark.gpu
def test_same_bits_every_time_and_in_a_graph():
    ts = tensors([1 << 18, 333, 70000, 5])
    out = [torch.empty_like(t) for t in ts]
    h.clip_grad_norm(ts, 0.5, out=out)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = h.clip_grad_norm(ts, 0.5, out=out)
    for i in range(4):
        for t, s in zip(ts, tensors([1 << 18, 333, 70000, 5], seed=i)):
            t.copy_(s)
        eager = [torch.empty_like(t) for t in ts]
        n = h.clip_grad_norm(ts, 0.5, out=eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_two_streams_at_once():
    a, b = tensors([1 << 20, 5]), tensors([300] * 40, seed=2)
    want = [h.grad_norm(a), h.grad_norm(b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for k, t in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                got[k] = h.grad_norm(t)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_a_tensor_of_several_pieces():
    """more elements than one entry of the kernel's table holds (2^30), the last ones alone in a second"""
    n = 2**30 + 4099
    t = torch.zeros(n, dtype=torch.float16, device="cuda")
    t[::1021], t[2**30 - 3:] = 0.5, 2.0
    small = torch.full((77,), 3.0, device="cuda")
    ones = (n + 1020) // 1021 - len(range(0, n, 1021)[(2**30 - 3 + 1020) // 1021:])
    norm = math.sqrt(0.25 * ones + 4.0 * (4099 + 3) + 9.0 * 77)
    got = h.clip_grad_norm([t, small], 1.0)
    assert abs(got.item() - norm) <= 2 * U * norm
    want = torch.zeros(n, dtype=torch.float16, device="cuda")
    want[::1021], want[2**30 - 3:] = t[0].item(), t[-1].item()
    assert torch.equal(t, want)
    check_clipped([t[:1], t[-1:], small], [torch.tensor([c / (norm + 1e-6)], dtype=torch.float64, device="cuda") for c in (0.5, 2.0, 3.0)])


# ---- refusals (no device is touched) -------------------------------------------------------------------------------------------------
def test_refusals():
    t = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="no tensors"):
        h.grad_norm([])
    with pytest.raises(ValueError, match="tensor 1 is not a float32"):
        h.grad_norm([t, t.double()])
    with pytest.raises(ValueError, match="tensor 0 is not a float32"):
        h.grad_norm([3.0])
    with pytest.raises(ValueError, match="tensor 0 is not contiguous"):
        h.grad_norm([t.t()])
    with pytest.raises(ValueError, match="overlap"):
        h.clip_grad_norm([t, t], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        h.clip_grad_norm([t[:3], t[2:]], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        h.clip_grad_norm([t[:2], t[2:]], 1.0, out=[torch.zeros(2, 6), t[:2]])
    with pytest.raises(ValueError, match="2 outputs for 1"):
        h.clip_grad_norm([t], 1.0, out=[t, t])
    with pytest.raises(ValueError, match="output 0 is torch.float32 of 12 elements"):
        h.clip_grad_norm([t], 1.0, out=[t[:2]])
    with pytest.raises(ValueError, match="output 0 is torch.float16"):
        h.clip_grad_norm([t], 1.0, out=[torch.zeros(4, 6, dtype=torch.float16)])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            h.clip_grad_norm([t], bad)
    with pytest.raises(h.MarlHipError, match="CPU"):
        h.clip_grad_norm([t], 1.0)


def test_c_entry_points_refuse():
    from codebase_amd import _lib

    tab = (_lib.TensorStruct * 1)(_lib.TensorStruct(None, None, 4, 0))
    assert _lib.lib.marlhip_grad_norm_workspace_bytes(tab, 1) < 0 and "tensor 0" in _lib.last_error()
    assert _lib.lib.marlhip_grad_norm_workspace_bytes(None, 1) < 0
    assert _lib.lib.marlhip_grad_norm_workspace_bytes(tab, -1) < 0
    tab[0] = _lib.TensorStruct(64, None, 4, 5)
    assert _lib.lib.marlhip_grad_norm_workspace_bytes(tab, 1) < 0 and "dtype" in _lib.last_error()
    tab[0] = _lib.TensorStruct(65, None, 4, 1)
    assert _lib.lib.marlhip_grad_norm_workspace_bytes(tab, 1) < 0 and "aligned" in _lib.last_error()
    tab[0] = _lib.TensorStruct(64, None, 4, 0)
    assert _lib.lib.marlhip_grad_norm(tab, 1, None, None, 0, None) < 0
    assert _lib.lib.marlhip_clip_grad_norm(tab, 1, float("nan"), 64, 64, 64, None) < 0 and "max_norm" in _lib.last_error()
