"""The batch's plan and what the batch functions refuse, on the CPU (a refused call launches nothing)."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from linuxformer_amd import seqs
from linuxformer_amd.seqs import Sequences, gated_delta, short_conv


def test_plan_tables():
    s = Sequences([130, 0, 1, 64], slots=[3, -1, 0, 5], device="cpu")
    t = s.tables.tolist()
    assert t == [[3, 0, 130, 0], [5, 131, 195, 4], [0, 130, 131, 3], [-1, 130, 130, 3],  # longest first
                 [0, 64, 0, 0], [64, 64, 0, 1], [128, 2, 0, 2], [130, 1, 2, 0], [131, 64, 1, 0]]
    assert (s.n_seqs, s.n_tokens, s.n_chunks, s.max_len, s.max_slot) == (4, 195, 5, 130, 5)
    e = Sequences([], device="cpu")
    assert (e.n_tokens, e.n_chunks, e.max_len, e.max_slot) == (0, 0, 0, -1)


@pytest.mark.parametrize("lengths,slots", [([1, -1], None), ([1, 2], [0]), ([1, 2], [4, 4]),
                                           ([1, 2], [0, -2]), ([1 << 31], None), ([1], [1 << 31])])
def test_plan_refuses(lengths, slots):
    with pytest.raises(ValueError):
        Sequences(lengths, slots, "cpu")


def _delta(N=5, nk=2, nv=4, K=64, V=32, dt=torch.bfloat16, slots=3):
    z = lambda *n, d=dt: torch.zeros(*n, dtype=d)  # noqa: E731
    return dict(q=z(N, nk, K), k=z(N, nk, K), v=z(N, nv, V), g=z(N, nv, d=torch.float32),
                beta=z(N, nv), state=z(slots, nv, K, V, d=torch.float32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(5, 2, 96, dtype=torch.bfloat16), k=torch.zeros(5, 2, 96, dtype=torch.bfloat16)),
    dict(k=torch.zeros(5, 2, 64)),
    dict(v=torch.zeros(5, 4, 24, dtype=torch.bfloat16)),
    dict(v=torch.zeros(5, 3, 32, dtype=torch.bfloat16)),
    dict(v=torch.zeros(4, 4, 32, dtype=torch.bfloat16)),
    dict(g=torch.zeros(5, 4, dtype=torch.float64)),
    dict(g=torch.zeros(5, 2)),
    dict(beta=torch.zeros(5, 4, dtype=torch.float16)),
    dict(state=torch.zeros(3, 4, 64, 32, dtype=torch.bfloat16)),
    dict(state=torch.zeros(3, 4, 32, 64).transpose(2, 3)),
    dict(state=torch.zeros(2, 4, 64, 32)),              # slot 2 is not there
    dict(state=torch.zeros(3 * 4 * 64 * 32 + 1)[1:].view(3, 4, 64, 32)),
    dict(state=torch.zeros(1, 4, 64, 32).expand(3, 4, 64, 32)),  # slots that share memory
    dict(out=torch.zeros(5, 4, 32)),
    dict(out=torch.zeros(5, 1, 32, dtype=torch.bfloat16).expand(5, 4, 32)),
    dict(seqs=Sequences([3, 3], device="cpu")),         # more tokens than rows
    dict(),                                             # nothing wrong, but no GPU
])
def test_gated_delta_refuses(change):
    a = dict(_delta(), seqs=Sequences([2, 0, 3], device="cpu"))
    a.update(change)
    with pytest.raises(ValueError) as e:
        gated_delta(**a)
    assert ("run on a GPU" in str(e.value)) == (not change), e.value


def test_gated_delta_refuses_gradients_and_takes_no_tokens():
    a = dict(_delta(), seqs=Sequences([5], device="cpu"))
    a["v"].requires_grad_()
    with torch.enable_grad(), pytest.raises(RuntimeError, match="gradients"):
        gated_delta(**a)
    a = dict(_delta(), seqs=Sequences([0, 0], device="cpu"))
    assert not gated_delta(**a).any()                   # (rows past the last sequence are zero)
    a["out"] = torch.full((5, 4, 32), 7.0, dtype=torch.bfloat16)
    assert (gated_delta(**a) == 7).all()                # and left as they were in out


@pytest.mark.parametrize("change", [
    dict(w=torch.zeros(8, 3)), dict(w=torch.zeros(8, 4, dtype=torch.float16)), dict(x=torch.zeros(5)),
    dict(x=torch.zeros(4, 8)), dict(window=torch.zeros(1, 8, 4)), dict(window=torch.zeros(2, 4, 8).mT),
    dict(window=torch.zeros(1, 8, 4).expand(2, 8, 4)),
    dict(x=torch.zeros(5, 8, dtype=torch.float64)), dict(out=torch.zeros(5, 4)), dict(),
])
def test_short_conv_refuses(change):
    a = dict(x=torch.zeros(5, 8), w=torch.zeros(8, 4), window=torch.zeros(2, 8, 4),
             seqs=Sequences([2, 3], device="cpu"))
    a.update(change)
    with pytest.raises(ValueError) as e:
        short_conv(**a)
    assert ("run on a GPU" in str(e.value)) == (not change), e.value


def test_scale_and_unit_are_read_at_each_call(monkeypatch):
    """A scale or a flag in a tensor that is changed between two calls."""
    seen = []
    monkeypatch.setattr(seqs, "_launch", lambda plan, f, table, io, *a: seen.append((io._obj.scale, io._obj.unit)))
    monkeypatch.setattr(seqs.mk_build, "load", lambda: SimpleNamespace(lxm_gd_recurrent=None))
    plan, scale, unit = Sequences([1], device="cpu"), torch.tensor(0.5), torch.tensor(True)
    a = [torch.zeros(s) for s in ((1, 1, 64), (1, 1, 64), (1, 1, 16), (1, 1), (1, 1), (1, 1, 64, 16))]
    gated_delta(*a, plan, scale=scale, unit=unit)
    scale.fill_(0.25), unit.fill_(False)
    gated_delta(*a, plan, scale=scale, unit=unit)
    assert seen == [(0.5, 1), (0.25, 0)]


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "state"])
def test_gated_delta_refuses_tangents(name):
    a = dict(_delta(), seqs=Sequences([5], device="cpu"))
    with torch.autograd.forward_ad.dual_level():
        a[name] = torch.autograd.forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match="gradients"):
            gated_delta(**a)
        with torch.no_grad(), pytest.raises(RuntimeError, match="gradients"):  # (tangents are formed there, too)
            gated_delta(**a)
        with torch.inference_mode(), pytest.raises(ValueError, match="run on a GPU"):  # (not here)
            gated_delta(**a)


@pytest.mark.parametrize("name", ["x", "w", "window"])
def test_short_conv_refuses_tangents(name):
    a = dict(x=torch.zeros(5, 8), w=torch.zeros(8, 4), window=torch.zeros(2, 8, 4), seqs=Sequences([2, 3], device="cpu"))
    with torch.autograd.forward_ad.dual_level():
        a[name] = torch.autograd.forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match="gradients"):
            short_conv(**a)


def test_an_out_that_needs_a_gradient_is_refused():
    a = dict(_delta(), seqs=Sequences([5], device="cpu"), out=torch.zeros(5, 4, 32, dtype=torch.bfloat16, requires_grad=True))
    c = dict(x=torch.zeros(5, 8), w=torch.zeros(8, 4), window=torch.zeros(2, 8, 4), seqs=Sequences([2, 3], device="cpu"),
             out=torch.zeros(5, 8, requires_grad=True))
    with torch.enable_grad():
        with pytest.raises(RuntimeError, match="gradients"):
            gated_delta(**a)
        with pytest.raises(RuntimeError, match="gradients"):
            short_conv(**c)
    with torch.no_grad(), pytest.raises(ValueError, match="run on a GPU"):
        gated_delta(**a)


@pytest.mark.parametrize("inference", [False, True])
def test_autograd_sees_what_is_written(monkeypatch, inference):
    """A cache or an out that something saved for its backward pass counts as changed (an inference tensor is never
    saved, and has no count)."""
    monkeypatch.setattr(seqs, "_launch", lambda *a: None)
    monkeypatch.setattr(seqs.mk_build, "load", lambda: SimpleNamespace(lxm_gd_recurrent=None, lxm_short_conv=None))
    plan = Sequences([1], device="cpu")
    with torch.inference_mode(inference):
        a = [torch.zeros(s) for s in ((1, 1, 64), (1, 1, 64), (1, 1, 16), (1, 1), (1, 1), (1, 1, 64, 16))]
        c = [torch.zeros(s) for s in ((1, 8), (8, 4), (1, 8, 4))]
        out, y = torch.zeros(1, 1, 16), torch.zeros(1, 8)
    gated_delta(*a, plan, out=out), short_conv(*c, plan, out=y)
    if inference:
        return
    assert [t._version for t in a + [out] + c + [y]] == [0, 0, 0, 0, 0, 1, 1, 0, 0, 1, 1]
    gated_delta(*a, plan), short_conv(*c, plan)
    assert [t._version for t in a + [out] + c + [y]] == [0, 0, 0, 0, 0, 2, 1, 0, 0, 2, 1]
    w = torch.ones(1, 1, 64, 16, requires_grad=True)
    with torch.enable_grad():
        loss = (w * a[5]).sum()
    gated_delta(*a, plan)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_an_out_whose_rows_overlap_is_refused():
    """Rows that reach into the next, in any order of the dimensions; views of a larger buffer do not."""
    plan, buf = Sequences([5], device="cpu"), torch.zeros(5, 6, 48)
    a = _delta(dt=torch.float32)
    for shape, strides in (((5, 4, 32), (64, 16, 1)), ((5, 4, 32), (16, 64, 1)), ((5, 4, 32), (128, 1, 1))):
        with pytest.raises(ValueError, match="share memory"):
            gated_delta(**a, seqs=plan, out=torch.as_strided(buf, shape, strides))
    for out in (buf[:, 1:5, 16:], buf.view(6, 5, 48).transpose(0, 1)[:, 2:, :32]):
        with pytest.raises(ValueError, match="run on a GPU"):
            gated_delta(**a, seqs=plan, out=out)
    c = dict(x=torch.zeros(5, 8), w=torch.zeros(8, 4), window=torch.zeros(1, 8, 4), seqs=plan)
    with pytest.raises(ValueError, match="share memory"):
        short_conv(**c, out=torch.as_strided(buf, (5, 8), (4, 1)))
    with pytest.raises(ValueError, match="run on a GPU"):
        short_conv(**c, out=buf[:, 0, :8])


def test_a_tensor_of_no_dimensions_is_refused():
    a = dict(_delta(), seqs=Sequences([5], device="cpu"), v=torch.zeros((), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        gated_delta(**a)
    with pytest.raises(ValueError):
        short_conv(torch.zeros(()), torch.zeros(8, 4), torch.zeros(1, 8, 4), Sequences([5], device="cpu"))


@pytest.mark.parametrize("change", [dict(K=96), dict(V=24), dict(V=272), dict(nk=0), dict(r=-1), dict(nk=70000), dict(type=3), dict()])
def test_workspace_of_what_is_not_allowed(native_lib, change):
    n = ctypes.c_int64(-1)
    e = native_lib.lxm_gd_ws(ctypes.byref(seqs.GdIO(**{**dict(nk=2, r=2, K=128, V=64, type=0), **change})), 3, ctypes.byref(n))
    assert (e, n.value) == (1, -1) if change else e == 0 and n.value > 0
