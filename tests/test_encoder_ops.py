"""The encoder operators' custom ops, which ``torch.compile`` calls, without a GPU: an eager call's
checks hold in the ops and in their fakes, where a bad argument is refused before any launch."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from torchwarp_b200.encoder import _ops

X, H, I, U = (2, 3, 8), torch.float16, torch.int64, torch.uint8
D = torch.float64

# t(shape, dtype): a tensor, real or a tracer's
CALLS = [
    (TypeError, lambda t: _ops.layer_norm(t(X, D), None, None, 1e-5)),
    (ValueError, lambda t: _ops.layer_norm(t((3, 0)), None, None, 1e-5)),
    (ValueError, lambda t: _ops.layer_norm(t(X), t((7,)), None, 1e-5)),
    (ValueError, lambda t: _ops.layer_norm(t(X), None, t((9,)), 1e-5)),
    (TypeError, lambda t: _ops.layer_norm(t(X), t((8,), H), None, 1e-5)),
    (TypeError, lambda t: _ops.layer_norm(t(X, H), t((8,)), t((8,), H), 1e-5)),
    (ValueError, lambda t: _ops.layer_norm(t(X), None, None, -1.0)),
    (ValueError, lambda t: _ops.layer_norm_backward(t((1, 3, 8)), t(X), None, None, t((2, 6)))),
    (ValueError, lambda t: _ops.layer_norm_backward(t(X), t(X), None, None, t((2, 5)))),
    (ValueError, lambda t: _ops.layer_norm_backward(t(X), t(X), None, None, t((2, 6), D))),
    (ValueError, lambda t: _ops.layer_norm_backward(t(X), t(X), t((7,)), None, t((2, 6)))),
    (TypeError, lambda t: _ops.linear(t(X, D), t((4, 8), D), None, None, 0)),
    (ValueError, lambda t: _ops.linear(t(X), t((4, 7)), None, None, 0)),
    (ValueError, lambda t: _ops.linear(t(X), t((8,)), None, None, 0)),
    (ValueError, lambda t: _ops.linear(t(X), t((4, 8)), t((3,)), None, 0)),
    (ValueError, lambda t: _ops.linear(t(X), t((4, 8)), None, t((2, 3, 1)), 0)),
    (TypeError, lambda t: _ops.linear(t(X), t((4, 8), H), None, None, 0)),
    (ValueError, lambda t: _ops.linear_backward(t((2, 3, 3)), t(X), t((4, 8)), t((0,)), 0)),
    (ValueError, lambda t: _ops.linear_backward(t((2, 3, 4)), t(X), t((4, 8)), t((5, 4)), 2)),
    (ValueError, lambda t: _ops.linear_backward(t((2, 3, 4)), t(X), t((4, 8)), t((6, 4), H), 2)),
    (TypeError, lambda t: _ops.gated_scan(t(X, D), t(X, D), None, None)),
    (ValueError, lambda t: _ops.gated_scan(t(X), t((2, 2, 8)), None, None)),
    (TypeError, lambda t: _ops.gated_scan(t(X), t(X, H), None, None)),
    (ValueError, lambda t: _ops.gated_scan(t(X), t(X), t((2, 7)), None)),
    (TypeError, lambda t: _ops.gated_scan(t(X), t(X), t((2, 8), H), None)),
    (ValueError, lambda t: _ops.gated_scan(t(X), t(X), None, t((3,), I))),
    (TypeError, lambda t: _ops.gated_scan(t(X), t(X), None, t((2,)))),
    (ValueError, lambda t: _ops.gated_scan_backward(t((1, 3, 8)), None, t(X), t(X), None,
                                                    t((64,), U))),
    (ValueError, lambda t: _ops.gated_scan_backward(None, t((2, 7)), t(X), t(X), None,
                                                    t((64,), U))),
    (ValueError, lambda t: _ops.gated_scan_backward(t(X), None, t(X), t(X), None, t((64,)))),
]


def real(shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def traced(shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("error,call", CALLS)
def test_refusals_of_the_ops(error, call):
    with pytest.raises(error):
        call(real)


@pytest.mark.parametrize("error,call", CALLS)
def test_refusals_while_tracing(error, call):
    with FakeTensorMode():
        with pytest.raises(error):
            call(traced)


@pytest.mark.parametrize("call", [
    lambda t: _ops.layer_norm(t(X), t((8,)), None, 1e-5),
    lambda t: _ops.linear(t(X), t((4, 8)), None, None, 0),
    lambda t: _ops.gated_scan(t(X), t(X), None, t((2,), I)),
])
def test_no_cpu_fallback_of_the_ops(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call(real)
    with FakeTensorMode():
        with pytest.raises(RuntimeError, match="CUDA"):
            call(real)


def test_devices_do_not_mix_while_tracing():
    with FakeTensorMode():
        x = torch.empty(2, 3, 8, device="cuda")
        for call in (lambda: _ops.layer_norm(x, torch.empty(8), None, 1e-5),
                     lambda: _ops.linear(x, torch.empty(4, 8), None, None, 0),
                     lambda: _ops.gated_scan(x, x, None, torch.empty(2, dtype=torch.int64))):
            with pytest.raises(RuntimeError):
                call()


def test_shapes_while_tracing():
    with FakeTensorMode():
        x, w = torch.empty(2, 3, 8, device="cuda"), torch.empty(4, 8, device="cuda")
        y, stats = _ops.layer_norm(x, None, None, 1e-5)
        assert y.shape == x.shape and stats.shape == (2, 6)
        y, z = _ops.linear(x, w, None, None, 2)
        assert y.shape == (2, 3, 4) and z.shape == (6, 4)
        y, state, _ = _ops.gated_scan(x, x, None, torch.empty(2, dtype=torch.int32, device="cuda"))
        assert y.shape == x.shape and state.shape == (2, 8) and state.dtype == torch.float32


def test_forward_mode_is_refused():
    """An eager call and the ops alike, whichever input has the tangent, also without gradients."""
    from torch.autograd import forward_ad
    import torchwarp_b200.functional as TF

    calls = [
        (lambda x, w, b: TF.layer_norm(x, w, b), [X, (8,), (8,)]),
        (lambda x, w, b, r: TF.linear(x, w, b, residual=r), [X, (4, 8), (4,), (2, 3, 4)]),
        (lambda x, g, h: TF.gated_scan(x, g, h), [X, X, (2, 8)]),
        (lambda x, g, h: TF.gated_scan_step(x, g, h), [(2, 8)] * 3),
        (lambda x, w, b: _ops.layer_norm(x, w, b, 1e-5), [X, (8,), (8,)]),
        (lambda x, w, b, r: _ops.linear(x, w, b, r, 0), [X, (4, 8), (4,), (2, 3, 4)]),
        (lambda x, g, h: _ops.gated_scan(x, g, h, None), [X, X, (2, 8)]),
    ]
    for call, shapes in calls:
        for which in range(len(shapes)):
            for grad in (False, True):
                with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    args = [real(s) for s in shapes]
                    args[which] = forward_ad.make_dual(args[which], torch.ones(shapes[which]))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(*args)


def test_tracers_see_the_operators():
    """Fake tensors and make_fx: shapes and graph nodes come from the ops, nothing is launched."""
    from torch.fx.experimental.proxy_tensor import make_fx
    import torchwarp_b200.functional as TF

    def f(x, w, b, r, g, h):
        y = TF.linear(TF.layer_norm(x, b), w, b, activation="gelu", residual=r)
        out, last = TF.gated_scan(y, g, h)
        return out, last, TF.gated_scan_step(y[:, 0], g[:, 0], h)

    shapes = [X, (8, 8), (8,), X, X, (2, 8)]
    with FakeTensorMode():
        out, last, y = f(*[traced(s) for s in shapes])
        assert out.shape == X and last.shape == (2, 8) and y.shape == (2, 8)
        args = [traced(s) for s in shapes]
    with torch.no_grad():
        graph = make_fx(f)(*args).graph
    names = [str(n.target) for n in graph.nodes if "torchwarp" in str(n.target)]
    assert names == ["torchwarp_b200.{}.default".format(n) for n in
                     ("layer_norm", "linear", "gated_scan", "gated_scan_step")]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_symbolic_lengths_stay_symbolic(dtype):
    """A dynamic time dimension is not fixed by the fakes, which give the sizes of the real ops."""
    from torch.fx.experimental.symbolic_shapes import (DimDynamic, ShapeEnv,
                                                       StatelessSymbolicContext)
    from torchwarp_b200 import _native

    env, plain = ShapeEnv(), torch.empty(3, 33, 20, dtype=dtype, device="meta")
    with FakeTensorMode(shape_env=env) as mode:
        dyn = StatelessSymbolicContext([DimDynamic.STATIC, DimDynamic.DYNAMIC, DimDynamic.STATIC])
        x = mode.from_tensor(plain, symbolic_context=dyn)
        x = torch.empty_like(x, device="cuda")
        w, n = traced((8, 20), dtype), traced((3,), I)
        assert isinstance(x.shape[1], torch.SymInt)
        _, stats = _ops.layer_norm(x, None, None, 1e-5)
        y, z = _ops.linear(x, w, None, None, 1)
        out, state, carry = _ops.gated_scan(x, x, None, n)
        dx, dg, dh = _ops.gated_scan_backward(out, state, x, x, n, carry)
        assert all(isinstance(v, torch.SymInt) for v in (stats.shape[1], y.shape[1], z.shape[0],
                                                         out.shape[1], carry.shape[0], dx.shape[1]))
    assert not env.replacements  # nothing fixed the symbol
    lib, size = _native.lib(), 4 if dtype == torch.float32 else 2
    for b, t, d in ((3, 33, 20), (1, 5000, 16), (1, 1, 1), (4, 0, 8), (2, 17, 8)):
        with FakeTensorMode():
            carry = _ops.gated_scan(traced((b, t, d), dtype), traced((b, t, d), dtype), None, None)[2]
        assert carry.numel() == (lib.tw_gated_scan_carry_bytes(b, t, d, size)
                                 - lib.tw_gated_scan_workspace_bytes(b, t, d, size))
