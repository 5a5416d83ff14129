"""The recurrent layer's operators where their inner loops run: pieces of many tokens, workgroups that walk many rows, steps that are taken as they are,
and gradients against differences.  Bounds are counted as in test_gpu_recurrent.py; a parameter's sum has as many additions behind one another as a
thread has tokens (a workgroup rows), a workgroup threads, and the last sum parts."""
import math

import pytest
import torch

from oracle import recurrent_oracle as O
from tests.test_gpu_recurrent import CONV_IN, NORM_IN, TYPES, _reference, _within, check_scan, norm_problem, run_conv, run_norm, run_scan, scan_problem

pytestmark = pytest.mark.gpu


def _code(kind):
    from rnn_train_ring_attractor_amd import _lib
    return _lib.load(), _lib.SEQUENCE_TYPES[TYPES[kind]]


# ------------------------------------------------------------------------------------------------
# What is not finite
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
def test_norm_of_gates_that_are_not_finite(kind, gpu_device):
    """NaN in a gate is NaN in y and, where the activation has a slope that depends on it, in the gate's own gradient, and the rest of the row is what it is without; a
    sigmoid of an infinite gate is one or zero, and its gradient zero."""
    dtype, C = TYPES[kind], 24
    for act in ("silu", "sigmoid", None):
        for value in (math.nan, math.inf, -math.inf):
            if act != "sigmoid" and not math.isnan(value):
                continue
            print(f"[case] gate {value} {act} {kind}", flush=True)
            p = norm_problem(59, (3,), C, dtype, next=False)
            clean = run_norm(p, dtype, gpu_device, group=8, activation=act)
            p["gate"][1, 5] = value
            got = run_norm(p, dtype, gpu_device, group=8, activation=act)
            rest = torch.ones(3, C, dtype=torch.bool, device=gpu_device)
            rest[1, 5] = False
            for n in ("y", "dgate"):
                assert torch.equal(got[n][rest], clean[n][rest]), (n, act, value)
                if math.isnan(value) and (n == "y" or act is not None):
                    assert torch.isnan(got[n][1, 5]), (n, act)
            if math.isnan(value):
                assert torch.isnan(got["dx"][1, :8]).all() and torch.equal(got["dx"][1, 8:], clean["dx"][1, 8:])
            else:
                p["gate"][1, 5] = 1e4 * math.copysign(1, value)
                want = run_norm(p, dtype, gpu_device, group=8, activation=act)
                assert all(torch.allclose(got[n], want[n], rtol=0, atol=1e-30) for n in ("y", "dgate", "dx"))


# ------------------------------------------------------------------------------------------------
# States over the borders of segments
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("A", [1.0, -1.0])
@pytest.mark.parametrize("what", ["nothing", "little", "much"])
def test_scan_across_powers_that_no_float_holds(what, A, kind, gpu_device):
    """Steps of one (of minus one, for a negative A that grows): over a segment of 96 tokens a state's power is e^96 or e^-96, which is infinite or zero in 32 bits.  A state of
    nothing stays nothing under it and 2^-100 becomes a number, as they do token by token; 2^100 under a negative A fades to one.  The same for the adjoint: inputs start
    behind the tokens whose outputs' gradients count, so that neither grows out of range.  Alone, and as one of 300 sequences, which are not cut."""
    dtype = TYPES[kind]
    for grows, T in ((True, 200), (False, 130)):
        step = 1.0 if (A > 0) == grows else -1.0
        if (what == "much") == grows:
            continue
        print(f"[case] powers {what} {A} {kind} {T}", flush=True)
        p = scan_problem(61, 1, T, 10, 5, 1, dtype, gate=False)
        first = {"nothing": 0.0, "little": 2.0 ** -100, "much": 2.0 ** 100}[what]
        p["A"], p["delta"], p["bias"] = torch.full_like(p["A"], A), torch.full_like(p["delta"], step), None
        late, early = (150, 50) if grows else (T, 0)
        p["x"][:, :late], p["dy"][:, early:] = 0, 0
        p["start"], p["de"] = first * p["start"].sign(), first * p["de"].sign()
        if grows and what == "little":           # (2^-100 e^200 is a number no longer: both end where x begins)
            T = 150
            p = {n: t[:, :T].contiguous() if n in ("x", "delta", "B", "C", "dy") else t for n, t in p.items()}
        got = run_scan(p, dtype, gpu_device, None, False)
        check_scan(p, got, None, False)
        shared = ("A", "D")
        many = run_scan({n: t if t is None or n in shared else t.expand(300, *t.shape[1:]) for n, t in p.items()}, dtype, gpu_device, None, False)
        size, total = O.scan_sizes(*(p[n] for n in ("x", "delta", "A", "B", "C", "D", "z", "bias", "start")), None, False, p["dy"], p["de"])
        for n in ("y", "state", "dx", "ddelta", "dB", "dC", "dstart"):
            assert torch.equal(many[n][299], many[n][0])
            a, b = got[n][0].double().cpu(), many[n][0].double().cpu()
            assert ((a - b).abs() <= torch.finfo(got[n].dtype).eps * b.abs() + 2 * (3 * T + 13 * total + 100) * 2.0 ** -24 * size[n][0] + 1e-37 + 1e-30 * (dtype == torch.float16))[
                torch.isfinite(b)].all() and (torch.isfinite(a) == torch.isfinite(b)).all(), n
