"""Host-side checks of the encoder operators that need no GPU: argument checks, the public names,
the C ABI's refusals and the missing CPU fallback."""

import copy
import pickle

import pytest
import torch

import torchwarp_b200 as tw
import torchwarp_b200.functional as TF
from torchwarp_b200 import _native


def test_public_names():
    for name in ("AdamW", "LayerNorm", "Linear", "EncoderBlock", "SequenceEncoder"):
        assert name in tw.__all__ and hasattr(tw, name)
    for name in ("layer_norm", "linear", "gated_scan", "gated_scan_step", "GatedScanOutput"):
        assert name in TF.__all__ and hasattr(TF, name)


X = torch.zeros(2, 3, 8)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: TF.layer_norm(X.double())),
    (TypeError, lambda: TF.layer_norm(X.long())),
    (ValueError, lambda: TF.layer_norm(torch.zeros(3, 0))),
    (ValueError, lambda: TF.layer_norm(torch.zeros(()))),
    (ValueError, lambda: TF.layer_norm(X, torch.ones(7))),
    (ValueError, lambda: TF.layer_norm(X, torch.ones(8), torch.ones(1, 8))),
    (TypeError, lambda: TF.layer_norm(X, torch.ones(8).half())),
    (TypeError, lambda: TF.layer_norm(X.half(), torch.ones(8), torch.ones(8).half())),
    (ValueError, lambda: TF.layer_norm(X, eps=-1.0)),
    (ValueError, lambda: TF.layer_norm(X, eps=float("nan"))),
    (TypeError, lambda: TF.layer_norm(X, None, None, 1e-5)),
    (TypeError, lambda: TF.linear(X.double(), torch.zeros(4, 8).double())),
    (ValueError, lambda: TF.linear(X, torch.zeros(4, 7))),
    (ValueError, lambda: TF.linear(X, torch.zeros(8))),
    (ValueError, lambda: TF.linear(X, torch.zeros(0, 8))),
    (ValueError, lambda: TF.linear(torch.zeros(2, 0), torch.zeros(4, 0))),
    (ValueError, lambda: TF.linear(X, torch.zeros(4, 8), torch.zeros(8))),
    (ValueError, lambda: TF.linear(X, torch.zeros(4, 8), residual=torch.zeros(2, 4))),
    (ValueError, lambda: TF.linear(X, torch.zeros(4, 8), residual=torch.zeros(2, 3, 1))),
    (TypeError, lambda: TF.linear(X, torch.zeros(4, 8).half())),
    (TypeError, lambda: TF.linear(X, torch.zeros(4, 8), residual=torch.zeros(2, 3, 4).half())),
    (ValueError, lambda: TF.linear(X, torch.zeros(4, 8), activation="tanh")),
    (TypeError, lambda: TF.gated_scan(X.double(), X.double())),
    (ValueError, lambda: TF.gated_scan(X[0], X[0])),
    (ValueError, lambda: TF.gated_scan(X, X[:, :2])),
    (TypeError, lambda: TF.gated_scan(X, X.half())),
    (ValueError, lambda: TF.gated_scan(X, X, torch.zeros(2, 7))),
    (TypeError, lambda: TF.gated_scan(X, X, torch.zeros(2, 8).half())),
    (ValueError, lambda: TF.gated_scan(X, X, lengths=torch.zeros(3, dtype=torch.int64))),
    (TypeError, lambda: TF.gated_scan(X, X, lengths=torch.zeros(2))),
    (ValueError, lambda: TF.gated_scan(torch.zeros(2, 3, 0), torch.zeros(2, 3, 0))),
    (ValueError, lambda: TF.gated_scan_step(X, X, torch.zeros(2, 8))),
    (ValueError, lambda: TF.gated_scan_step(X[0], X[0], None)),
    (TypeError, lambda: TF.gated_scan_step(X[0], X[0], torch.zeros(3, 8).double())),
    (ValueError, lambda: TF.gated_scan_step(X[0], X[0], torch.zeros(8, 3).t())),
    (ValueError, lambda: tw.Linear(4, 4, activation="tanh")),
])
def test_refusals(error, call):
    with pytest.raises(error):
        call()


def _params():
    return [torch.nn.Parameter(torch.zeros(4))]


@pytest.mark.parametrize("kw", [{"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)},
                                {"eps": -1.0}, {"weight_decay": -0.1}, {"state_bits": 16}])
def test_adamw_refusals(kw):
    with pytest.raises(ValueError):
        tw.AdamW(_params(), **kw)


@pytest.mark.parametrize("call", [
    lambda: TF.layer_norm(X),
    lambda: TF.linear(X, torch.zeros(4, 8)),
    lambda: TF.gated_scan(X, X),
    lambda: TF.gated_scan_step(X[0], X[0], torch.zeros(3, 8)),
    lambda: tw.SequenceEncoder(8, 16)(X),
    lambda: tw.AdamW(_params()).step(),
])
def test_no_cpu_fallback(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


def test_c_abi_refusals_without_a_gpu():
    """Argument errors come back as a status and a message, before any launch."""
    lib = _native.lib()
    p = 256  # never dereferenced: the call is refused first
    assert lib.tw_layer_norm_forward_f32(p, 4, p, p, 0, 2, 0, 1e-5, p, None, None, None) == 1
    assert lib.tw_layer_norm_forward_f32(None, 4, p, p, 0, 2, 4, 1e-5, p, None, None, None) == 1
    assert lib.tw_layer_norm_forward_f32(p, 4, p, p, 0, 2, 4, -1.0, p, None, None, None) == 1
    assert lib.tw_layer_norm_forward_f32(p, 4, p, p, 0, 2, 4, 1e-5, p, p, None, None) == 1
    assert lib.tw_layer_norm_forward_f32(p, 4, p, p, 0, 0, 4, 1e-5, p, None, None, None) == 0
    assert lib.tw_linear_forward_bf16(p, 8, p, 8, None, None, 0, 2, 0, 8, 0, p, None, None, 0,
                                      None) == 1
    assert lib.tw_linear_forward_bf16(p, 8, p, 8, None, None, 0, 2, 4, 8, 9, p, None, None, 0,
                                      None) == 1
    assert lib.tw_linear_forward_bf16(p, 8, None, 8, None, None, 0, 2, 4, 8, 0, p, None, None, 0,
                                      None) == 1
    assert lib.tw_linear_backward_f32(p, 4, p, 8, p, 8, None, 2, 4, 8, 3, p, p, p, p, 1 << 40,
                                      None) == 1
    assert lib.tw_linear_backward_f32(p, 4, p, 8, p, 8, p, 2, 4, 8, 3, p, p, p, p, 0, None) == 5
    assert lib.tw_gated_scan_forward_f16(p, 8, 8, p, 8, 8, None, None, -1, 2, 8, p, p, None, 0,
                                         None) == 1
    assert lib.tw_gated_scan_forward_f16(p, 8, 8, p, 8, 8, None, None, 1, 2, 8, p, None, None, 0,
                                         None) == 1
    assert lib.tw_gated_scan_forward_f16(p, 8, 8, p, 8, 8, None, None, 1, 2, 8, p, p, p, 0,
                                         None) == 5
    assert lib.tw_gated_scan_step_f32(p, 8, p, 8, None, 1, 8, p, None) == 1
    assert lib.tw_adamw_step_f32(p, 1, 16, p, None, p, None, p, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, 0,
                                 None) == 1
    assert lib.tw_adamw_step_f32(p, 1, 8, p, None, p, None, p, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, 0,
                                 None) == 1
    assert lib.tw_adamw_step_f32(p, 1, 32, p, None, p, None, None, 1e-3, None, 0.9, 0.99, 1e-8, 0.0,
                                 0, None) == 1
    assert lib.tw_adamw_step_f32(p, 1, 32, p, None, p, None, p, 1e-3, None, 1.0, 0.99, 1e-8, 0.0,
                                 0, None) == 1
    assert b"beta" in lib.tw_last_error()


@pytest.mark.parametrize("again", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_adamw_is_copied_whole(again):
    opt = again(tw.AdamW(_params(), lr=0.5, state_bits=8, seed=7))
    assert (opt._bits, opt._seed, opt.param_groups[0]["lr"]) == (8, 7, 0.5)
    with pytest.raises(RuntimeError, match="CUDA"):
        opt.step()
