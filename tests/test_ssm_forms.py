"""The state space operators' forms against the 64-bit definition: lanes a channel, whole and split sequences, single steps, stretches of the
convolution, rows that a wave takes one after the other.  Tolerances as in test_ssm.py, whose references these are."""
import pytest
import torch

from codebase_amd import hip as h
from tests.test_ssm import check_scan, make_scan, scan_call, scan_grad_call


def name_of(shape):
    return "x".join(map(str, shape))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 24, 16, 66, 16, 1), (1, 24, 16, 40, 8, 1), (1, 24, 16, 40, 3, 1), (1, 24, 1040, 66, 8, 1), (1, 24, 1040, 66, 16, 1), (1, 24, 16, 66, 32, 1),
                                   (1, 192, 16, 66, 16, 1)], ids=name_of)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gradients_just_before_a_reset(shape, bad):
    """row b ends an episode with a state that is not finite at step b mod 16, wherever that lies in a block of steps: the gradient of that step's output
    map says so, and every other step's is as finite as the state it is multiplied with"""
    P, S, B, C, N, G = shape
    v = make_scan(*shape, reset=False, lengths=False)
    rows = torch.arange(B, device="cuda")
    last = rows % 16
    v["x"] = v["x"].clone()
    v["x"][:, last, rows] = bad
    v["reset"] = torch.zeros(S, B, dtype=torch.uint8, device="cuda")
    v["reset"][last + 1, rows] = 1
    record = h.ssm_scan_record(v["x"], N)
    y = scan_call(v, record=record)
    g = scan_grad_call(v, record)
    at = torch.zeros(S, B, dtype=torch.bool, device="cuda")
    at[last, rows] = True
    assert not torch.isfinite(y[:, at]).any() and bool(torch.isfinite(y[:, ~at]).all())
    assert not torch.isfinite(g.C[:, at]).any()
    assert bool(torch.isfinite(g.C[:, ~at]).all()) and bool(torch.isfinite(g.x).all()) and bool(torch.isfinite(g.A).all())


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1024, 2048])  # 16 chunks and 32: joined in one go and in runs
def test_empty_states_in_sequences_that_grow(S):
    """a state of 0 stays 0 whatever it is multiplied with, and so does a gradient: 128 steps by e^16 each, past any float's range"""
    v = make_scan(1, S, 1, 20, 4, z=False, bias=False, softplus=False, lengths=False)
    step = torch.arange(S, device="cuda")[None, :, None, None]
    late, early = step >= S - 148, step < 200
    v["A"], v["h_in"], v["dh_out"] = torch.ones_like(v["A"]), None, None
    v["reset"] = late[0, :, :, 0].logical_and(step[0, :, :, 0] == S - 148).to(torch.uint8)
    grow = torch.where((step >= 256) & (step < 384), 16.0, 0.0).expand_as(v["x"])
    # empty up to the reset, an episode behind it
    w = dict(v, x=torch.where(late, v["x"], 0.0), dy=torch.where(late, v["dy"], 0.0), delta=torch.where(late, 0.01, grow))
    y, hT, g = check_scan(w)
    assert hT.any() and y.any() and g.x.any()
    # gradients in front of the growth, none behind it
    w = dict(v, x=torch.zeros_like(v["x"]), dy=torch.where(early, v["dy"], 0.0), delta=torch.where(early, 0.01, grow))
    _, _, g = check_scan(w)
    assert g.x.any()


def test_sizes_beyond_the_c_structs_are_refused():
    x, w = torch.zeros(2, 1, 1, 4), torch.zeros(2, 4, 4)
    for call in (lambda: h.ssm_conv(x[:1].expand(1, 1, 2**31, 4), w[:1]), lambda: h.ssm_scan_record(x, 2**31), lambda: h.ssm_conv(x, w, sharing=(0, 1.0))):
        with pytest.raises(ValueError, match="not 32-bit integers"):
            call()
    with pytest.raises(ValueError, match="one per agent"):
        h.ssm_conv(x[:0], w, sharing=())
