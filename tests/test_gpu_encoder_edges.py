"""The encoder operators where inputs, tensors or programs are unlike a plain eager call (B200)."""

import copy
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def tw():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import torchwarp_b200
    return torchwarp_b200


@pytest.fixture(autouse=True, scope="module")
def _no_device_error():
    yield
    if torch.cuda.is_available():
        from torchwarp_b200 import _native
        assert _native.lib().tw_device_error() == 0


@pytest.fixture
def randn():
    g = torch.Generator(device=DEV).manual_seed(0)
    return lambda *shape, dtype=torch.float32: torch.randn(*shape, device=DEV,
                                                           generator=g).to(dtype)


# ------------------------------------------------------------ compiled calls

def test_compiled_calls_take_strided_parameters(tw, randn):
    TF = tw.functional
    x, gate = randn(4, 30, 16), randn(4, 30, 16)
    w, nw, nb, b = randn(16, 16), randn(32)[::2], randn(32)[1::2], randn(48)[::3]
    lengths = torch.tensor([30, 0, 7, 0, 29, 0, 1, 0], device=DEV)[::2]

    def f(x, gate):
        y = TF.linear(TF.layer_norm(x, nw, nb), w, b, activation="silu")
        return TF.gated_scan(y, gate, lengths=lengths)

    torch._dynamo.reset()
    want, got = f(x, gate), torch.compile(f, fullgraph=True, backend="aot_eager")(x, gate)
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
    for kind in (torch.int32, torch.int64):
        torch._dynamo.reset()
        n = lengths.to(kind)
        out = torch.compile(lambda x, g: TF.gated_scan(x, g, lengths=n), backend="aot_eager")(x, gate)
        assert torch.equal(out.output, TF.gated_scan(x, gate, lengths=lengths).output)


def test_compiled_calls_refuse_bad_arguments(tw, randn):
    """While the function is traced: nothing is launched."""
    TF = tw.functional
    x = randn(4, 30, 16)
    for f in (lambda x: TF.layer_norm(x, x.new_ones(15)), lambda x: TF.linear(x, x.new_ones(8, 17)),
              lambda x: TF.linear(x, x.new_ones(8, 16), residual=x.new_ones(4, 1, 8)),
              lambda x: TF.gated_scan(x, x[:, :1]),
              lambda x: TF.gated_scan(x, x, lengths=torch.zeros(4, dtype=torch.int64))):
        torch._dynamo.reset()
        with pytest.raises(Exception, match="must (have|be)|CUDA"):
            torch.compile(f, fullgraph=True, backend="aot_eager")(x)


# ------------------------------------------------------------------- AdamW

def _stepped(tw, randn, sizes, **kw):
    ps = [torch.nn.Parameter(randn(n)) for n in sizes]
    for p in ps:
        p.grad = randn(p.numel())
    opt = tw.AdamW(ps, **kw)
    opt.step()
    return ps, opt


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_refuses_other_parameters_than_its_states(tw, randn, bits):
    """A replaced, added, dropped, longer or shorter parameter: nothing is written."""
    def refused(change, back):
        ps, opt = _stepped(tw, randn, [300, 40, 7], state_bits=bits)
        was = [v.clone() for v in opt.flat_state().values()]
        group = opt.param_groups[0]["params"]
        values = [p.detach().clone() for p in group]
        change(group)
        with pytest.raises(ValueError):
            opt.step()
        back(group, ps)
        for v, w in zip(opt.flat_state().values(), was):
            assert torch.equal(v.float(), w.float())
        for p, v in zip(ps, values):
            assert torch.equal(p.detach(), v)
        opt.step()

    def put(group, ps):
        group[:] = ps

    def resize(n):
        def change(group):
            group[0].grad = None
            group[0].data = randn(n)
            group[0].grad = randn(n)
        return change

    new = torch.nn.Parameter(randn(40))
    new.grad = randn(40)
    refused(lambda g: g.__setitem__(1, new), put)
    refused(lambda g: g.append(new), put)
    refused(lambda g: g.pop(), put)
    refused(lambda g: g.reverse(), put)
    for n in (4000, 301, 299, 0):
        ps, opt = _stepped(tw, randn, [300, 40, 7], state_bits=bits)
        was = [v.clone() for v in opt.flat_state().values()]
        resize(n)(ps)
        with pytest.raises(ValueError):
            opt.step()
        for v, w in zip(opt.flat_state().values(), was):
            assert torch.equal(v.float(), w.float())


def test_adamw_takes_new_groups_later(tw, randn):
    ps, opt = _stepped(tw, randn, [300])
    new = torch.nn.Parameter(randn(5))
    new.grad = randn(5)
    opt.add_param_group({"params": [new], "lr": 1e-2})
    was = new.detach().clone()
    kept = opt.flat_state(0)["exp_avg"].clone()
    ps[0].grad = None
    opt.step()
    # a first step moves a weight by lr along its gradient's sign
    torch.testing.assert_close(new.detach(), was * (1 - 1e-4) - 1e-2 * new.grad.sign())
    assert torch.equal(opt.flat_state(0)["exp_avg"], kept)


# ------------------------------------------------------------------ linear

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("m", [4, 200])
def test_linear_slopes_where_the_saved_z_is_infinite(tw, randn, m, act, dtype):
    """z past the type's largest value is saved as an infinity; the slope there is 0 or 1.
    Tolerances: those of tests/test_gpu_encoder.py for gradients, 4 roundings to the type and 64
    of float32 in the 2-norm."""
    big = {torch.float16: 7e4, torch.bfloat16: 3.395e38, torch.float32: 1e30}[dtype]
    unit = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}[dtype]
    k = 16
    x, w = randn(m, k) * 0.5, randn(24, k) * 0.25
    x[:, 0], x[1, 0], w[:, 0], w[0, 0], w[1, 0] = 0, 64, 0, -big / 64, big / 64
    x, w = (v.to(dtype).requires_grad_(True) for v in (x, w))
    dy = randn(m, 24, dtype=dtype)
    grads = torch.autograd.grad(tw.functional.linear(x, w, activation=act), (x, w), dy)
    xd, wd = x.detach().double(), w.detach().double()
    z = xd @ wd.t()
    assert float(z[1, 1]) > 0.9 * big and float(z[1, 0]) < -0.9 * big
    if act == "relu":
        slope = (z > 0).double()
    elif act == "gelu":
        slope = torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * 0.3989422804014327
    else:
        f = torch.sigmoid(z)
        slope = f * (1 + z * (1 - f)) if act == "silu" else f * (1 - f)
    dz = dy.double() * slope
    # the columns of w that hold `big` meet dx alone: compare the others, and that those are finite
    for got, want in zip(grads, (dz @ wd, dz.t() @ xd)):
        assert torch.isfinite(got).all() or dtype != torch.float16
        got, want = got.double()[:, 1:], want[:, 1:]
        err, bound = float((got - want).norm()), (4 * unit + 64 * 2.0 ** -24) * float(want.norm())
        assert err <= bound + 2.0 ** -24 * want.numel() ** 0.5, (err, bound)


# ------------------------------------------------------ tracers, transforms

def _program(tw, randn):
    TF = tw.functional
    w, b = randn(32, 32) / 6, randn(32)

    def f(x, gate, lengths, w, b):
        y = TF.linear(TF.layer_norm(x, b), w, b, activation="gelu", residual=x)
        out, last = TF.gated_scan(y, gate, lengths=lengths)
        return out, last

    def args(*t):
        return randn(3, 20, 32), randn(3, 20, 32), torch.tensor(t, device=DEV), w, b
    return f, args


def test_traced_programs_compute(tw, randn):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, args = _program(tw, randn)
    a, b = args(20, 3, 7), args(5, 20, 0)
    want = f(*b)
    for program in (torch.jit.trace(f, a), make_fx(f)(*a), make_fx(f, tracing_mode="fake")(*a),
                    make_fx(f, tracing_mode="symbolic")(*a)):
        for got, w in zip(program(*b), want):
            assert torch.equal(got, w)

    def stream(x, gate, state):
        return tw.functional.gated_scan_step(x, gate, state)

    s = [randn(4, 32) for _ in range(3)]
    for trace in (lambda: torch.jit.trace(stream, [v.clone() for v in s], check_trace=False),
                  lambda: make_fx(stream)(*[v.clone() for v in s])):
        program = trace()
        x, gate, state = (randn(4, 32) for _ in range(3))
        other = state.clone()
        assert torch.equal(program(x, gate, state), stream(x, gate, other))
        assert torch.equal(state, other)


def test_dispatch_modes_and_subclasses(tw, randn):
    """An operator under a mode gives the bits and the gradients of a plain call."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))

    f, args = _program(tw, randn)
    x, *rest = args(20, 3, 7)
    x.requires_grad_(True)
    want = f(x, *rest)[0]
    wg, = torch.autograd.grad(want.sum(), x)
    names = []
    with Log():
        got = f(x, *rest)[0]
        gg, = torch.autograd.grad(got.sum(), x)
    for name in ("layer_norm", "linear", "gated_scan"):
        assert "torchwarp_b200.{}.default".format(name) in names
        assert "torchwarp_b200.{}_backward.default".format(name) in names
    assert torch.equal(got, want) and torch.equal(gg, wg)


def test_function_transforms(tw, randn):
    """vmap goes slice by slice; derivatives by torch.func, which the operators lack, raise."""
    f, args = _program(tw, randn)
    x, *rest = args(20, 3, 7)
    with pytest.raises(Exception):
        torch.func.grad(lambda x: f(x, *rest)[0].square().sum())(x)
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: f(x, *rest)[0], (x,), (x,))
    for got, want in zip(torch.func.vmap(f, (0, 0, 0, None, None))(
            *(torch.stack([v, v.flip(0)]) for v in (x, *rest[:2])), *rest[2:]), f(x, *rest)):
        assert torch.equal(got[0], want) and torch.equal(got[1], want.flip(0))


def test_compiled_forward_mode_is_refused(tw, randn):
    from torch.autograd import forward_ad
    x = randn(2, 20, 32)
    for f in (lambda x: tw.functional.layer_norm(x), lambda x: tw.functional.linear(x, x[0, :4]),
              lambda x: tw.functional.gated_scan(x, x).output):
        def level(x):
            with forward_ad.dual_level():
                return forward_ad.unpack_dual(f(forward_ad.make_dual(x, x))).tangent
        for g in (lambda x: torch.func.jvp(f, (x,), (x,))[1], level):
            torch._dynamo.reset()
            with pytest.raises(Exception, match="forward-mode"):
                torch.compile(g, backend="aot_eager")(x)
        torch._dynamo.reset()  # and a call after it compiles
        assert torch.equal(torch.compile(f, backend="aot_eager", fullgraph=True)(x), f(x))


def test_compiled_stream(tw, randn):
    """A frame of a live stream in one compiled graph: eager's bits, the states updated in place."""
    torch._dynamo.reset()
    enc = tw.SequenceEncoder(5, 32, layers=2, device=DEV)
    step = torch.compile(enc.step, fullgraph=True, backend="aot_eager")
    a, b = enc.init_state(3), enc.init_state(3)
    for _ in range(4):
        x = randn(3, 5)
        got, want = step(x, a), enc.step(x, b)
        assert torch.equal(got, want)
        for u, v in zip(a, b):
            assert torch.equal(u, v)
    x = randn(3, 16).requires_grad_(True)
    with pytest.raises(Exception, match="not differentiable"):
        torch.compile(tw.functional.gated_scan_step, backend="aot_eager")(x, x, randn(3, 16))


def test_compiled_once_for_all_lengths(tw, randn):
    """Time marked dynamic: one graph, right at every length, forward and backward."""
    from torch._dynamo.testing import CompileCounterWithBackend
    TF = tw.functional
    w, b = randn(48, 24), randn(48)

    def f(x):
        v, a = TF.linear(TF.layer_norm(x), w, b, activation="silu").split(24, -1)
        return TF.gated_scan(v, a).output

    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    g = torch.compile(f, backend=counter, fullgraph=True)
    for t in (33, 700, 5, 129, 2000):
        x = randn(3, t, 24).requires_grad_(True)
        torch._dynamo.mark_dynamic(x, 1)
        got = g(x)
        dx, = torch.autograd.grad(got.square().sum(), x)
        want = f(x)
        wx, = torch.autograd.grad(want.square().sum(), x)
        assert torch.equal(got, want) and torch.equal(dx, wx)
    assert counter.frame_count == 1


def test_compiled_inference_saves_nothing(tw, randn):
    """What only a backward needs is written when one can follow, not in a call without gradients."""
    TF = tw.functional
    x, w = randn(3, 40, 32), randn(64, 32)

    def f(x, w):
        v, a = TF.linear(TF.layer_norm(x), w, activation="gelu").split(32, -1)
        return TF.gated_scan(v, a)

    def saves(x, w, grad):
        graphs = []

        def backend(gm, inputs):
            graphs.append(gm)
            return gm.forward

        torch._dynamo.reset()
        with torch.set_grad_enabled(grad):
            got, want = torch.compile(f, backend=backend, fullgraph=True)(x, w), f(x, w)
        assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
        return [n.args[-1] for n in graphs[0].graph.nodes if "torchwarp" in str(n.target)]

    assert saves(x, w, True) == [False] * 3 and saves(x, w.requires_grad_(True), False) == [False] * 3
    assert saves(x, w, True) == [False, True, True]
    ops = torch.ops.torchwarp_b200
    assert ops.layer_norm(x, None, None, 1e-5, False)[1].numel() == 0
    assert ops.linear(x, w.detach(), None, None, 2, False)[1].numel() == 0
    assert ops.gated_scan(x, x, None, None, False)[2].numel() == 0
    # a backward without what it needs is refused
    with pytest.raises(ValueError):
        ops.layer_norm_backward(x, x, None, None, ops.layer_norm(x, None, None, 1e-5, False)[1])
    with pytest.raises(ValueError):
        ops.linear_backward(randn(3, 40, 64), x, w.detach(), randn(0), 2)
    with pytest.raises(RuntimeError):
        ops.gated_scan_backward(x, None, x, x, None, torch.empty(0, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("again", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_adamw_copies_go_on_by_themselves(tw, randn, bits, again):
    """A copy has its own weights and states, and takes the steps that the optimizer takes."""
    ps, opt = _stepped(tw, randn, [300, 5], state_bits=bits, seed=4)
    ps.append(torch.nn.Parameter(randn(40).half()))
    ps[-1].grad = randn(40).half()
    opt.add_param_group({"params": ps[-1:]})
    opt.step()
    other = again(opt)
    qs = [p for g in other.param_groups for p in g["params"]]
    for p, q in zip(ps, qs):
        assert p is not q and torch.equal(p, q)
        q.grad = p.grad.clone()
    for _ in range(2):
        opt.step()
    for p, q in zip(ps, qs):
        assert not torch.equal(p, q)
    for _ in range(2):
        other.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    for k in range(2):
        for a, b in zip(opt.flat_state(k).values(), other.flat_state(k).values()):
            assert a.data_ptr() != b.data_ptr() and torch.equal(a.float(), b.float())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_steps_without_gradients_do_not_count(tw, randn, bits):
    """The first step that has a gradient is the first: it moves a weight by lr."""
    p = torch.nn.Parameter(randn(300))
    opt = tw.AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
    for _ in range(3):
        opt.step()
    was, p.grad = p.detach().clone(), randn(300)
    opt.step()
    torch.testing.assert_close(p.detach(), was - 1e-2 * p.grad.sign(), rtol=1e-5, atol=1e-6)
    p.grad, was = None, p.detach().clone()
    opt.step()
    assert torch.equal(p, was) and opt.state_dict()["buckets"][0]["step"].tolist() == [1]


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_refused_checkpoints_change_nothing(tw, randn, bits):
    _, opt = _stepped(tw, randn, [300, 7], state_bits=bits, lr=1e-2, seed=1)
    _, longer = _stepped(tw, randn, [600, 7], state_bits=bits, lr=1.0, seed=2)
    _, fewer = _stepped(tw, randn, [300], state_bits=bits, lr=1.0, seed=2)
    _, other = _stepped(tw, randn, [300, 7], state_bits=40 - bits, lr=1.0, seed=2)
    short = _stepped(tw, randn, [300, 7], state_bits=bits, lr=1.0, seed=2)[1].state_dict()
    del short["buckets"][0]["step"]
    was = copy.deepcopy(opt.state_dict())
    for bad in (longer.state_dict(), fewer.state_dict(), other.state_dict(), short):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        now = opt.state_dict()
        assert now["param_groups"] == was["param_groups"] and now["seed"] == 1
        for a, b in zip(now["buckets"], was["buckets"]):
            assert all(torch.equal(a[k].float(), b[k].float()) for k in b)


def test_adamw_state_dict_is_one_moment(tw, randn):
    """The step count follows the states of the same dictionary; a copy keeps both."""
    ps, opt = _stepped(tw, randn, [300])
    live, kept = opt.state_dict(), copy.deepcopy(opt.state_dict())
    weights = [p.detach().clone() for p in ps]
    opt.step()
    after = [p.detach().clone() for p in ps]
    assert live["buckets"][0]["step"].item() == 2 and kept["buckets"][0]["step"].item() == 1
    assert torch.equal(live["buckets"][0]["exp_avg"], opt.flat_state()["exp_avg"])
    for p, w in zip(ps, weights):
        p.detach().copy_(w)
    opt.load_state_dict(kept)
    opt.step()
    assert all(torch.equal(p, a) for p, a in zip(ps, after))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adamw_8_bit_bad_gradients_stay_in_their_place(tw, randn, dtype):
    """An infinite or NaN gradient spoils its own weight, not the 255 whose scale it shares: they
    take the bits that they take when it is zero."""
    bad = {3: float("inf"), 40: float("-inf"), 41: float("nan"), 700: float("inf"), 899: float("nan")}
    start = randn(900, dtype=dtype)
    grads = [randn(900, dtype=dtype) * 1e-2 for _ in range(3)]
    for g in grads:
        g[list(bad)] = 0

    def run(first):
        p = torch.nn.Parameter(start.clone())
        opt = tw.AdamW([p], lr=1e-2, state_bits=8, seed=9)
        for g in [first] + grads[1:]:
            p.grad = g
            opt.step()
        return p.detach(), opt.flat_state()

    wrong = grads[0].clone()
    for k, v in bad.items():
        wrong[k] = v
    (p, s), (q, t) = run(wrong), run(grads[0])
    fine = torch.ones(900, dtype=torch.bool, device=DEV)
    fine[list(bad)] = False
    assert torch.isnan(p[~fine]).all() and torch.equal(p[fine], q[fine])
    for k in s:
        if k.endswith("scale"):
            assert torch.equal(s[k], t[k])
        else:
            a, b = s[k].float()[:900], t[k].float()[:900]
            assert torch.isnan(a[~fine]).all() and torch.equal(a[fine], b[fine])


# ------------------------------------------------------ windows of a signal

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,hop", [(64, 16), (64, 1), (33, 8), (400, 160), (9000, 512)])
def test_overlapping_rows(tw, randn, size, hop, dtype):
    """Windows as a view of their signal give what a copy of them gives."""
    TF = tw.functional
    rows = randn(2, 30 * hop + size, dtype=dtype).unfold(-1, size, hop)
    w, b = randn(size, dtype=dtype), randn(size, dtype=dtype)
    lw = (randn(24, size) / size ** 0.5).to(dtype)
    for f in (lambda x: TF.layer_norm(x, w, b), lambda x: TF.linear(x, lw, activation="silu")):
        view, dense = (v.detach().requires_grad_(True) for v in (rows, rows.contiguous()))
        assert view.stride(1) == hop
        y, want = f(view), f(dense)
        dy = randn(*y.shape, dtype=dtype)
        dx, = torch.autograd.grad(y, view, dy)
        wx, = torch.autograd.grad(want, dense, dy)
        # alignment may choose another form of a kernel: 16 roundings of float32, one to the type
        unit = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -20
        for got, ref in ((y.detach(), want.detach()), (dx, wx)):
            assert float((got.float() - ref.float()).norm()) <= unit * float(ref.float().norm())


# ---------------------------------------------------------------- autocast

@pytest.mark.parametrize("compiled", [False, True])
def test_autocast_casts_what_torch_casts(tw, randn, compiled):
    torch._dynamo.reset()
    f = tw.functional.linear
    if compiled:
        f = torch.compile(f, backend="aot_eager")
    x, w, b = randn(20, 32), randn(8, 32), randn(8)
    with torch.autocast("cuda", torch.bfloat16):
        y = f(x, w.half(), b)
        assert torch.equal(y, tw.functional.linear(x.bfloat16(), w.half().bfloat16(), b.bfloat16()))
        for bad in ((x.double(), w), (x, w.double()), (x.long(), w), (x, w, b.double())):
            torch._dynamo.reset()
            with pytest.raises(Exception, match="must be"):
                f(*bad)
    leaf = w.clone().requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16):  # a weight used twice
        loss = (f(x, leaf, b).float() + f(2 * x, leaf, b).float()).sum()
    dw, = torch.autograd.grad(loss, leaf)
    want = 3 * x.bfloat16().float().sum(0).expand(8, 32)
    assert dw.dtype == torch.float32
    # each of the two gradients, and their sum, is rounded to bfloat16
    torch.testing.assert_close(dw, want, rtol=2.0 ** -6, atol=2.0 ** -6)


# --------------------------------------------------------------- infinities

def _same_but_rounding(got, want, unit):
    """NaN and infinities in the same places, the rest within `unit` of the largest of its row."""
    got, want = got.detach().double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    for sign in (1, -1):
        assert torch.equal(got == sign * float("inf"), want == sign * float("inf"))
    fine = torch.isfinite(want)
    zero = torch.zeros_like(want)
    err = torch.where(fine, got - want, zero).abs()
    assert (err <= unit * torch.where(fine, want, zero).abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(2, 64, 96), (8, 20, 33), (300, 64, 96), (20, 40, 4096),
                                   (17, 129, 65), (700, 512, 256)])
def test_linear_infinities_follow_the_definition(tw, randn, m, n, k, dtype):
    """inf w is an infinity of w's sign, inf 0 and inf - inf are NaN, whatever the number of rows.
    Rounding: one to the type (2^-8, 2^-11) and a few of float32 in sums of like terms."""
    inf = float("inf")
    x, w = randn(m, k, dtype=dtype), (randn(n, k) / k ** 0.5).to(dtype)
    dy = randn(m, n, dtype=dtype)
    x[1, 3], w[5, 3] = inf, 0
    if m > 8:
        x[7, 0], x[7, k - 1] = inf, -inf
        x[9, 20] = float("nan")
        w[11, 21], dy[13, 2] = -inf, inf
    w[:, 1], x[0, 0] = w[:, 1].sign() * 0.5, 1  # one bfloat16 plane each
    x.requires_grad_(True)
    w.requires_grad_(True)
    unit = {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[dtype]
    y = tw.functional.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xd, wd, dyd = (v.detach().double().cpu() for v in (x, w, dy))

    def product(a, b):
        """a b^T by the definition: sums that hold infinities are the sum of those."""
        out = torch.where(torch.isfinite(a), a, 0.0) @ torch.where(torch.isfinite(b), b, 0.0).t()
        for i in range(len(a)):
            if not torch.isfinite(a[i]).all():
                out[i] = (a[i] * b).sum(1)
        for j in range(len(b)):
            if not torch.isfinite(b[j]).all():
                out[:, j] = (a * b[j]).sum(1)
        return out.to(DEV)

    _same_but_rounding(y, product(xd, wd), unit)
    _same_but_rounding(dx, product(dyd, wd.t()), unit)
    _same_but_rounding(dw, product(dyd.t(), xd.t()), unit)


def _scan_by_definition(x, gate, h0, lengths, dy, dstate):
    """f h + (1 - f) x and its adjoints in 64 bits; past its length a sequence keeps its state, has
    outputs and gradients 0, and what it holds there is not read."""
    t = x.shape[1]
    live = (torch.arange(t, device=DEV) < lengths.unsqueeze(1)).unsqueeze(2)
    x, f, dy = (torch.where(live, v.double(), 0.0) for v in (x, gate, dy))
    f = torch.sigmoid(f)
    omf = torch.sigmoid(-torch.where(live, gate.double(), 0.0))
    h, hs = h0.double(), []
    for k in range(t):
        hs.append(h)
        h = torch.where(live[:, k], f[:, k] * h + omf[:, k] * x[:, k], h)
    y = torch.where(live, torch.stack(hs[1:] + [h], 1), 0.0)
    last, lam = h, dstate.double()
    dx, dg = torch.zeros_like(x), torch.zeros_like(x)
    for k in range(t - 1, -1, -1):
        on = live[:, k]
        l = lam + dy[:, k]
        dx[:, k] = torch.where(on, omf[:, k] * l, 0.0)
        dg[:, k] = torch.where(on, l * (hs[k] - x[:, k]) * f[:, k] * omf[:, k], 0.0)
        lam = torch.where(on, f[:, k] * l, lam)
    return y, last, dx, dg, lam


# sizes that reach each form of the scan: segments of time, blocks of a cluster (rows off 16 bytes),
# one block, half lines, whole lines, a warp alone
SCAN_FORMS = [(2, 700, 16), (1, 5000, 64), (1, 5000, 3), (3, 300, 33), (40, 130, 97), (5, 700, 2048),
              (40, 700, 96), (5, 300, 2048), (29, 203, 1000), (32, 97, 1024)]


def _scan_inputs(randn, b, t, d, dtype, mean=2.0):
    lengths = torch.tensor([(t, 0, 1, t - 1, t // 3)[k % 5] for k in range(b)], device=DEV)
    u = randn(b, t, 2 * d)
    u[..., d:] = u[..., d:] * 1.5 + mean
    x, gate = u.to(dtype).split(d, -1)
    return x, gate, randn(b, d), lengths, randn(b, t, d, dtype=dtype), randn(b, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,t,d", SCAN_FORMS)
def test_scan_infinities_follow_the_definition(tw, randn, b, t, d, dtype):
    """An infinite state stays one, at live frames and past a sequence's length."""
    inf = float("inf")
    x, gate, h0, lengths, dy, ds = _scan_inputs(randn, b, t, d, dtype)
    h0[:, 0], h0[0, 1], ds[:, 2 % d] = inf, -inf, inf
    x[0, t // 2, 1 % d], x[0, 40, 2 % d], x[0, 60, 2 % d] = inf, -inf, inf
    x[0, 33, d - 1], dy[0, 90, d // 2] = float("nan"), -inf
    x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
    h0.requires_grad_(True)
    y, last = tw.functional.gated_scan(x, gate, h0, lengths=lengths)
    grads = torch.autograd.grad((y, last), (x, gate, h0), (dy, ds))
    want = _scan_by_definition(*(v.detach() for v in (x, gate, h0)), lengths, dy, ds)
    assert torch.isinf(want[1]).any() and torch.isinf(want[2]).any()
    unit = {torch.float32: 2.0 ** -16, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[dtype]
    for got, w in zip((y, last) + grads, want):
        _same_but_rounding(got, w, unit)


def test_scan_infinite_state_through_closed_gates(tw, randn):
    """Products of small gates that underflow keep an infinity; a gate of -inf does not."""
    for d in (8, 5):
        x, h0 = randn(3, 200, d), torch.full((3, d), float("inf"), device=DEV)
        gate = torch.full((3, 200, d), -20.0, device=DEV)
        gate[1, 50], gate[2, 199] = float("-inf"), float("-inf")
        y, last = tw.functional.gated_scan(x, gate, h0)
        assert torch.isinf(y[0]).all() and torch.isinf(last[0]).all()
        assert torch.isinf(y[1, :50]).all() and torch.isnan(y[1, 50:]).all()
        assert torch.isinf(y[2, :199]).all() and torch.isnan(last[2]).all()


def test_scan_step_infinities(tw, randn):
    state, x, gate = randn(4, 8), randn(4, 8), randn(4, 8)
    state[0], state[1], x[2], x[1, 0] = float("inf"), float("-inf"), float("inf"), float("inf")
    want = torch.sigmoid(gate) * state + torch.sigmoid(-gate) * x
    y = tw.functional.gated_scan_step(x, gate, state)
    _same_but_rounding(y, want, 2.0 ** -20)
    _same_but_rounding(state, want, 2.0 ** -20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("b,t,d", SCAN_FORMS)
def test_scan_forms(tw, randn, b, t, d, ragged, dtype):
    """Each form over several tiles and a partial last one, whole and with lengths of 0, 1, T - 1
    and inside a tile.  Tolerances: one rounding to the type and 64 of float32, in the 2-norm, and
    float16's smallest step."""
    x, gate, h0, lengths, dy, ds = _scan_inputs(randn, b, t, d, dtype)
    if not ragged:
        lengths.fill_(t)
    x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
    h0.requires_grad_(True)
    y, last = tw.functional.gated_scan(x, gate, h0, lengths=lengths if ragged else None)
    grads = torch.autograd.grad((y, last), (x, gate, h0), (dy, ds))
    want = _scan_by_definition(*(v.detach() for v in (x, gate, h0)), lengths, dy, ds)
    for got, w in zip((y, last) + grads, want):
        unit = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[got.dtype]
        err = float((got.detach().double() - w).norm())
        floor = 2.0 ** -24 * w.numel() ** 0.5 if got.dtype == torch.float16 else 0.0
        assert err <= (unit + 64 * 2.0 ** -24) * float(w.norm()) + floor
    with torch.no_grad():
        y2, last2 = tw.functional.gated_scan(x, gate, h0, lengths=lengths if ragged else None)
    assert torch.equal(y, y2) and torch.equal(last, last2)


@pytest.mark.parametrize("m", [1, 20])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("least,most", [(-104, 20), (-6, 6), (-8, 5.9)])
def test_float32_activation_tails(tw, least, most, m, act):
    """Far from 0 the small side of silu and sigmoid keeps float32's relative precision, into its
    subnormals: an exponential of 2 ulp, a sum, a division and a product of half an ulp each, 8
    spacings of 2^-23 allowed; below 2^-126 the spacing is 2^-149.  z is the bias, and its gradient,
    a sum before any product, is dz."""
    z = torch.linspace(least, most, 300, device=DEV)
    leaf = z.clone().requires_grad_(True)
    zero = torch.zeros(m, 4, device=DEV)
    y = tw.functional.linear(zero, torch.zeros(300, 4, device=DEV), leaf, activation=act)
    dy = torch.zeros_like(y)
    dy[0] = 1
    dz, = torch.autograd.grad(y, leaf, dy)
    assert (y == y[0]).all()
    y = y[0]
    f, omf = torch.sigmoid(z.double()), torch.sigmoid(-z.double())
    if act == "silu":
        want, slope = z.double() * f, f * (1 + z.double() * omf)
        near = (1 + z.double() * omf).abs() > 0.1  # where the slope's factor does not cancel
    else:
        want, slope, near = f, f * omf, torch.ones_like(f, dtype=torch.bool)
    for got, w, where in ((y.detach(), want, torch.ones_like(near)), (dz, slope, near)):
        bound = 8 * 2.0 ** -23 * w.abs() + 104 * 2.0 ** -149
        # the slope's factor and the large side of f add their own roundings
        bound = bound if w is want else 8 * bound
        assert ((got.double() - w).abs() <= bound)[where].all()


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_states_are_float32_whatever_the_default_type(tw, randn, default):
    x = randn(3, 20, 5)
    results = []
    for kind in (torch.float32, default):
        torch.manual_seed(1)
        enc = tw.SequenceEncoder(5, 16, layers=1, device=DEV, dtype=torch.float32)
        torch.set_default_dtype(kind)
        try:
            states = enc.init_state(3)
            y = enc.step(x[:, 0], states)
            out = [y, *states]
            for bits in (8, 32):
                opt = tw.AdamW(enc.parameters(), state_bits=bits)
                enc(x).square().sum().backward()
                opt.step()
                out += [v for k, v in opt.flat_state().items()]
                for k, v in opt.flat_state().items():
                    assert v.dtype == (torch.float8_e4m3fn if bits == 8 and "scale" not in k
                                       else torch.float32)
        finally:
            torch.set_default_dtype(torch.float32)
        results.append([v.float() for v in out] + [p.detach() for p in enc.parameters()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_adamw_step_refuses_states_of_another_kind(tw, randn):
    """The host entry itself: nothing is launched on buffers that the kernel would overrun."""
    from torchwarp_b200 import _native
    p = torch.nn.Parameter(randn(600))
    p.grad = randn(600)
    f = dict(device=DEV, dtype=torch.float32)
    m, s, step = torch.zeros(768, **f), torch.zeros(3, **f), torch.zeros(2, device=DEV,
                                                                       dtype=torch.int32)
    c = torch.zeros(768, device=DEV).to(torch.float8_e4m3fn)
    rest = (step, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 0)
    host = _native.host()
    host.adamw_step([p], [600], 32, m, None, m.clone(), None, *rest)
    host.adamw_step([p], [600], 8, c, s, c.clone(), s.clone(), *rest)
    for bits, a, x, b, y in ((32, m.bfloat16(), None, m, None), (32, m, None, m.double(), None),
                             (32, m[:767], None, m, None), (32, m, s, m, s), (32, m.cpu(), None, m, None),
                             (8, c, s, m, s), (8, c, s[:2], c, s), (8, c, None, c, s),
                             (8, c, s, c, s.bfloat16())):
        with pytest.raises((RuntimeError, ValueError)):
            host.adamw_step([p], [600], bits, a, x, b, y, *rest)


def test_adamw_first_step_is_not_captured(tw, randn):
    """A graph that made the states would zero them at every replay."""
    p = torch.nn.Parameter(randn(300))
    p.grad = randn(300)
    opt = tw.AdamW([p], lr=1e-2)
    was = p.detach().clone()
    with pytest.raises(RuntimeError, match="before a step is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p, was)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(2):
        graph.replay()
    assert opt.state_dict()["buckets"][0]["step"].item() == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,d", SCAN_FORMS)
def test_scan_bad_values_stay_in_their_channel(tw, randn, b, t, d, dtype):
    """Every other channel, and in time all that a bad value does not reach, keeps its bits."""
    x, gate, h0, lengths, dy, ds = _scan_inputs(randn, b, t, d, dtype)
    c, at = (0, d - 1), t // 2

    def run(spoil):
        xs, hs, ys, es = x.clone(), h0.clone(), dy.clone(), ds.clone()
        if spoil:
            xs[0, at, c[0]], xs[0, at, c[1]] = float("nan"), float("inf")
            hs[2 % b, 0], ys[0, at, d // 2], es[0, 1] = float("-inf"), float("nan"), float("inf")
        leaves = [v.requires_grad_(True) for v in (xs, gate.detach().clone(), hs)]
        y, last = tw.functional.gated_scan(*leaves, lengths=lengths)
        return y, last, *torch.autograd.grad((y, last), leaves, (ys, es))

    spoilt = torch.zeros(b, d, dtype=torch.bool, device=DEV)
    spoilt[0, [0, d - 1, d // 2, 1]] = True
    spoilt[2 % b, 0] = True
    got, want = run(True), run(False)
    for u, w in zip(got, want):
        u, w = (v.transpose(1, 2) if v.dim() == 3 else v for v in (u, w))
        assert torch.equal(u[~spoilt], w[~spoilt])
    assert torch.equal(got[0][0, :at, d - 1], want[0][0, :at, d - 1])  # outputs before a bad input


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("m,n,k", [(4, 64, 32), (200, 130, 96), (20, 40, 4096)])
def test_linear_values_do_not_depend_on_their_neighbours(tw, randn, m, n, k, act, dtype):
    """Large, infinite and NaN values in some columns leave the bits of the others."""
    x, w, b = randn(m, k, dtype=dtype), (randn(n, k) / k ** 0.5).to(dtype), randn(n, dtype=dtype)
    want = tw.functional.linear(x, w, b, activation=act)
    odd = torch.zeros(n, dtype=torch.bool, device=DEV)
    odd[[0, 5, 9, 33]] = True
    b[0], b[5], b[9], b[33] = 50, -90, float("inf"), float("nan")
    got = tw.functional.linear(x, w, b, activation=act)
    assert torch.equal(got[:, ~odd], want[:, ~odd])


def test_adamw_refused_step_changes_nothing(tw, randn):
    """With several types and groups, what the last of them refuses holds the first back too."""
    a, b = (torch.nn.Parameter(randn(40, 30, dtype=t)) for t in (torch.bfloat16, torch.float32))
    c = torch.nn.Parameter(randn(7))
    opt = tw.AdamW([{"params": [a, b]}, {"params": [c]}])
    for p in (a, b, c):
        p.grad = randn(*p.shape, dtype=p.dtype)
    opt.step()

    def held_back():
        was = [p.detach().clone() for p in (a, b, c)]
        steps = [s["step"].item() for s in opt.state_dict()["buckets"]]
        with pytest.raises(ValueError):
            opt.step()
        assert all(torch.equal(p, w) for p, w in zip((a, b, c), was))
        assert [s["step"].item() for s in opt.state_dict()["buckets"]] == steps == [1, 1, 1]

    b.data = randn(30, 40).t()  # no longer contiguous
    held_back()
    b.data = randn(40, 30)
    opt.param_groups[1]["lr"] = torch.ones(2, device=DEV)
    held_back()
    opt.param_groups[1]["lr"] = 1e-3
    c.grad, c.data = None, randn(9)
    c.grad = randn(9)
    held_back()
