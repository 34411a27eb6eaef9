"""The encoder operators on a B200 against plain 64-bit forms.

Tolerances.  u = 2^-24, 2^-8, 2^-11 is half a spacing of float32, bfloat16, float16 (relative).
An output of 16 bits is rounded once, so its 2-norm error is at most u of its type beside the
float32 error of what was rounded.  The float32 stage is allowed 64 roundings of 2^-24 (3.8e-6 in
the 2-norm): sums are split over lanes and tiles, so no chain of dependent additions of like signs
is longer than that in effect.  A linear layer's 16-bit gradients go through z and dz, each rounded
to 16 bits: 3 u in all, 4 u allowed.  Differences are central, with step h: h^2 truncation and
2 * 64 u / h rounding, both below 2e-3 at h = 2^-5 for these smooth functions.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 64 * 2.0 ** -24
DEV = "cuda"


@pytest.fixture(scope="module")
def TF():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import torchwarp_b200.functional as TF
    return TF


@pytest.fixture(autouse=True, scope="module")
def _no_device_error():
    yield
    if torch.cuda.is_available():
        from torchwarp_b200 import _native
        assert _native.lib().tw_device_error() == 0


def rng(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, g, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def close(got, want, rounds=1.0, floor=0.0, extra=1.0):
    """2-norm error within `rounds` roundings to got's type and the float32 allowance; `floor` is
    an absolute part (float16 subnormals, cancelled results)."""
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all()
    got, u = got.double(), U[got.dtype]
    err = float((got - want).norm())
    bound = (rounds * u + extra * F32) * float(want.norm()) + floor * math.sqrt(max(want.numel(), 1))
    assert err <= bound, (err, bound, float(want.norm()))


# ------------------------------------------------------------- layer norm

def ln_plain(x, w, b, eps, dy=None):
    x, w, b = (None if t is None else t.double() for t in (x, w, b))
    w = torch.ones_like(x[0]) if w is None else w
    mu = x.mean(-1, keepdim=True)
    xc = x - mu
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    y = xh * w + (0 if b is None else b)
    if dy is None:
        return y
    dy = dy.double()
    q = dy * w
    dx = rstd * (q - q.mean(-1, keepdim=True) - xh * (q * xh).mean(-1, keepdim=True))
    return y, dx, (dy * xh).sum(0), dy.sum(0)


LN_SHAPES = [(1, 1), (1, 256), (3, 7), (2, 2), (5, 257), (17, 1024), (130, 768), (4, 8192), (2, 20000),
             (1000, 8), (4097, 33), (700, 500), (1, 40000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim", LN_SHAPES)
def test_layer_norm(TF, rows, dim, dtype):
    g = rng(rows * 7 + dim)
    x = (randn(rows, dim, g=g) * 2 + randn(rows, 1, g=g)).to(dtype).requires_grad_(True)
    w = (1 + 0.1 * randn(dim, g=g)).to(dtype).requires_grad_(True)
    b = (0.1 * randn(dim, g=g)).to(dtype).requires_grad_(True)
    dy = randn(rows, dim, g=g, dtype=dtype)
    y = TF.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    wy, wdx, wdw, wdb = ln_plain(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    # dx of few columns is a difference that cancels to the size of eps: an absolute part in
    # units of dy * rstd (below 400 here)
    floor = 400 * F32 if dim <= 8 else 0.0
    close(y.detach(), wy)
    close(dx, wdx, floor=floor)
    close(dw, wdw, floor=F32)
    close(db, wdb)
    with torch.no_grad():
        assert torch.equal(TF.layer_norm(x, w, b), y)  # the form without statistics
        again = TF.layer_norm(x, w, b)
    assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(TF, dtype, weight, bias):
    g = rng(3)
    x = randn(2, 9, 100, g=g, dtype=dtype).requires_grad_(True)
    w = randn(100, g=g).requires_grad_(True) if weight else None  # float32 parameters
    b = randn(100, g=g).requires_grad_(True) if bias else None
    dy = randn(2, 9, 100, g=g, dtype=dtype)
    y = TF.layer_norm(x, w, b, eps=1e-3)
    live = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, live, dy)
    wy, wdx, wdw, wdb = ln_plain(x.detach().view(18, 100), w if w is None else w.detach(),
                                 b if b is None else b.detach(), 1e-3, dy.view(18, 100))
    want = [wdx.view(2, 9, 100)] + ([wdw] if weight else []) + ([wdb] if bias else [])
    close(y.detach(), wy.view(2, 9, 100))
    for got, wnt, leaf in zip(grads, want, live):
        assert got.dtype == leaf.dtype
        close(got, wnt)


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_strides(TF, dtype):
    g = rng(4)
    base = randn(64, 300, g=g, dtype=dtype)
    w, b = randn(128, g=g, dtype=dtype), randn(128, g=g, dtype=dtype)
    flat = randn(64 * 128 + 3, g=g, dtype=dtype)
    for x in (base[:, :128], base[:, 5:133], base[:, :256:2], base.t()[:128, :].t(),
              flat[1:1 + 64 * 128].view(64, 128), flat[3:].view(64, 128),
              base[:1, :128].expand(64, 128), base[::2, 40:168]):
        for dy in (randn(*x.shape, g=g, dtype=dtype), randn(*x.shape, g=g, dtype=dtype)[:1].expand(x.shape)):
            xl = x.detach().requires_grad_(True)
            y = TF.layer_norm(xl, w, b)
            dx, = torch.autograd.grad(y, xl, dy)
            wy, wdx, _, _ = ln_plain(x, w, b, 1e-5, dy)
            close(y.detach(), wy)
            close(dx, wdx)


def test_layer_norm_offset_and_constant_rows(TF):
    g = rng(5)
    x = randn(8, 512, g=g) + 4096.0  # the mean loses 12 bits, the variance must not lose 24
    y = TF.layer_norm(x)
    close(y, ln_plain(x, None, None, 1e-5), floor=4096 * 2.0 ** -24 * 4)
    c = torch.full((3, 512), 7.0, device=DEV)
    assert torch.equal(TF.layer_norm(c), torch.zeros_like(c))
    b = randn(512, g=g)
    assert torch.equal(TF.layer_norm(c, None, b), b.expand(3, 512))


def test_layer_norm_bad_values_stay_in_their_row(TF):
    x = randn(6, 130, g=rng(6))
    x[2, 5], x[4, 0] = float("nan"), float("inf")
    y = TF.layer_norm(x)
    ok = [0, 1, 3, 5]
    assert torch.isfinite(y[ok]).all() and torch.isnan(y[[2, 4]]).all()


def test_layer_norm_empty(TF):
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    y = TF.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w))


# ----------------------------------------------------------------- linear

ACTS = [None, "relu", "gelu", "silu", "sigmoid"]


def act_plain(z, act):
    if act == "relu":
        return torch.relu(z), (z > 0).double()
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        f = torch.sigmoid(z)
        return z * f, f * (1 + z * (1 - f))
    if act == "sigmoid":
        f = torch.sigmoid(z)
        return f, f * (1 - f)
    return z, torch.ones_like(z)


def linear_plain(x, w, b, r, act, dy=None):
    x, w = x.double(), w.double()
    z = x @ w.t() + (0 if b is None else b.double())
    y, s = act_plain(z, act)
    if r is not None:
        y = y + r.double()
    if dy is None:
        return y
    dz = dy.double() * s
    return y, dz @ w, dz.t() @ x, dz.sum(0)


def linear_case(TF, m, n, k, dtype, act, seed=0, bias=True, residual=False, extra=1.0):
    g = rng(seed + m + 3 * n + 5 * k)
    x = randn(m, k, g=g, dtype=dtype).requires_grad_(True)
    w = (randn(n, k, g=g) / math.sqrt(k)).to(dtype).requires_grad_(True)
    b = (0.1 * randn(n, g=g)).to(dtype).requires_grad_(True) if bias else None
    r = randn(m, n, g=g, dtype=dtype).requires_grad_(True) if residual else None
    dy = randn(m, n, g=g, dtype=dtype)
    y = TF.linear(x, w, b, activation=act, residual=r)
    live = [t for t in (x, w, b, r) if t is not None]
    grads = dict(zip([k_ for k_, t in zip("xwbr", (x, w, b, r)) if t is not None],
                     torch.autograd.grad(y, live, dy)))
    d = [None if t is None else t.detach() for t in (x, w, b, r)]
    if act == "relu":
        # its slope near 0 is decided by the last bits of z: keep clear of it
        z = d[0].double() @ d[1].double().t() + (0 if b is None else d[2].double())
        far = z.abs() > 64 * (2.0 ** -24 + U[dtype]) * math.sqrt(k)
        dy = dy * far
        grads = dict(zip(grads, torch.autograd.grad(TF.linear(x, w, b, activation=act, residual=r),
                                                    live, dy)))
    wy, wdx, wdw, wdb = linear_plain(*d, act, dy)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    close(y.detach(), wy, extra=extra, floor=tiny)
    close(grads["x"], wdx, 4, extra=extra, floor=tiny)
    close(grads["w"], wdw, 4, extra=extra, floor=tiny * math.sqrt(m))
    if bias:
        close(grads["b"], wdb, 4, extra=extra, floor=tiny * math.sqrt(m))
    if residual:
        assert torch.equal(grads["r"], dy)
    with torch.no_grad():
        assert torch.equal(TF.linear(x, w, b, activation=act, residual=r), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 64, 64), (3, 5, 7), (8, 256, 128), (17, 129, 65), (64, 384, 257), (128, 128, 64),
    (129, 130, 131), (200, 56, 84), (1000, 72, 1024), (1, 1000, 2048), (5, 8, 4096), (2049, 16, 40),
    (300, 512, 512), (16, 1024, 1024), (33, 2000, 24), (4096, 256, 64)])
def test_linear_sizes(TF, m, n, k, dtype):
    linear_case(TF, m, n, k, dtype, "silu", residual=(m + n) % 2 == 0, bias=k % 3 != 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [4, 190])
def test_linear_activations(TF, act, m, dtype):
    linear_case(TF, m, 96, 160, dtype, act, seed=1)
    linear_case(TF, m, 96, 160, dtype, act, seed=2, bias=False, residual=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [6, 200])
def test_linear_strides(TF, m, dtype):
    g = rng(8)
    wide = randn(m, 400, g=g, dtype=dtype)
    odd = randn(m * 128 + 1, g=g, dtype=dtype)[1:].view(m, 128)
    w0 = (randn(96, 128, g=g) / 11).to(dtype)
    wt = (randn(128, 96, g=g) / 11).to(dtype).t()
    ww = (randn(96, 300, g=g) / 11).to(dtype)
    r0 = randn(m, 300, g=g, dtype=dtype)
    for x in (wide[:, :128], wide[:, 8:136], wide[:, 3:131], odd, wide[:1, :128].expand(m, 128),
              wide.t()[:128].t()):
        for w in (w0, wt, ww[:, :128], ww[:, 1:129]):
            for r in (r0[:, :96], r0[:, 5:101]):
                xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
                y = TF.linear(xl, wl, None, activation="gelu", residual=r)
                dy = randn(m, 200, g=g, dtype=dtype)[:, 7:103]
                dx, dw = torch.autograd.grad(y, (xl, wl), dy)
                wy, wdx, wdw, _ = linear_plain(x, w, None, r, "gelu", dy)
                close(y.detach(), wy)
                close(dx, wdx, 4)
                close(dw, wdw, 4)


def test_linear_leading_dimensions_and_empty(TF):
    g = rng(9)
    x = randn(2, 3, 5, 40, g=g).requires_grad_(True)
    w = randn(24, 40, g=g).requires_grad_(True)
    y = TF.linear(x, w)
    assert y.shape == (2, 3, 5, 24)
    close(y.detach().view(30, 24), linear_plain(x.detach().view(30, 40), w.detach(), None, None, None))
    e = torch.zeros(0, 40, device=DEV, requires_grad=True)
    dx, dw = torch.autograd.grad(TF.linear(e, w, activation="silu"), (e, w), torch.zeros(0, 24, device=DEV))
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("m", [2, 300])
def test_linear_bad_values_stay_in_their_row(TF, m):
    for dtype in TYPES:
        x, w = randn(m, 96, g=rng(1), dtype=dtype), randn(64, 96, g=rng(2), dtype=dtype)
        x[1, 3] = float("inf")
        y = TF.linear(x, w)
        keep = torch.arange(m, device=DEV) != 1
        assert torch.isfinite(y[keep]).all() and not torch.isfinite(y[1]).any()


def test_linear_float32_precision(TF):
    """float32 products keep float32: a long contraction of positive terms."""
    g = rng(10)
    x, w = torch.rand(300, 8192, device=DEV, generator=g), torch.rand(200, 8192, device=DEV, generator=g)
    close(TF.linear(x, w), linear_plain(x, w, None, None, None))


# ------------------------------------------------------------ gated scan

def scan_plain(x, gate, h0, lengths, dy=None, dstate=None):
    x, f = x.double(), torch.sigmoid(gate.double())
    b, t, d = x.shape
    h = torch.zeros(b, d, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    n = [t] * b if lengths is None else [max(0, min(t, int(v))) for v in lengths]
    live = torch.tensor([[k < v for k in range(t)] for v in n], device=x.device).view(b, t, 1)
    f = torch.where(live, f, torch.ones_like(f))
    x = torch.where(live, x, torch.zeros_like(x))
    hs = [h]
    for k in range(t):
        hs.append(f[:, k] * hs[-1] + (1 - f[:, k]) * x[:, k])
    y = torch.stack(hs[1:], 1) * live if t else x
    if dy is None and dstate is None:
        return y, hs[-1]
    dy = torch.zeros_like(x) if dy is None else torch.where(live, dy.double(), torch.zeros_like(x))
    lam = torch.zeros_like(h) if dstate is None else dstate.double()
    dx, dg = torch.zeros_like(x), torch.zeros_like(x)
    for k in range(t - 1, -1, -1):
        lam = lam + dy[:, k]
        dx[:, k] = (1 - f[:, k]) * lam
        dg[:, k] = lam * (hs[k] - x[:, k]) * f[:, k] * (1 - f[:, k])
        lam = f[:, k] * lam
    return y, hs[-1], dx, dg, lam


def scan_case(TF, b, t, d, dtype, lengths=None, with_state=True, use=(True, True), mean=2.0):
    g = rng(b + 3 * t + 7 * d)
    u = randn(b, t, 2 * d, g=g)
    u[..., d:] = u[..., d:] * 1.5 + mean
    u = u.to(dtype)
    x, gate = (v.detach().requires_grad_(True) for v in u.split(d, -1))  # strided halves
    h0 = randn(b, d, g=g).requires_grad_(True) if with_state else None
    dy = randn(b, t, d, g=g, dtype=dtype) if use[0] else None
    ds = randn(b, d, g=g) if use[1] else None
    if lengths is not None:
        lengths = torch.tensor(lengths, device=DEV)
        with torch.no_grad():
            for k, v in enumerate(lengths.tolist()):  # what is masked is never read
                x[k, max(0, v):] = float("nan")
                gate[k, max(0, v):] = float("inf")
                if dy is not None:
                    dy[k, max(0, v):] = float("nan")
    y, last = TF.gated_scan(x, gate, h0, lengths=lengths)
    live = [v for v in (x, gate, h0) if v is not None]
    outs = [(o, go) for o, go in ((y, dy), (last, ds)) if go is not None]
    grads = torch.autograd.grad([o for o, _ in outs], live, [go for _, go in outs])
    wy, wl, wdx, wdg, wdh = scan_plain(x.detach(), gate.detach(), None if h0 is None else h0.detach(),
                                       lengths, dy, ds)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    assert last.dtype == torch.float32
    close(y.detach(), wy, floor=tiny)
    close(last.detach(), wl, floor=tiny)
    for got, want in zip(grads, (wdx, wdg, wdh)):
        close(got, want, floor=tiny)
    with torch.no_grad():
        y2, l2 = TF.gated_scan(x, gate, h0, lengths=lengths)
    assert torch.equal(y, y2) and torch.equal(last, l2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,d", [
    (1, 1, 1), (2, 2, 3), (1, 31, 8), (3, 32, 64), (2, 33, 65), (4, 100, 256), (1, 1000, 24),
    (2, 2500, 16), (1, 257, 1000), (5, 7, 2048), (40, 65, 96), (1, 5000, 2)])
def test_scan_sizes(TF, b, t, d, dtype):
    scan_case(TF, b, t, d, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [40, 700])
def test_scan_lengths(TF, t, dtype):
    scan_case(TF, 7, t, 48, dtype, lengths=[t, 0, 1, t - 1, 33, t + 9, -3])
    scan_case(TF, 3, t, 20, dtype, lengths=[0, 0, 0])


@pytest.mark.parametrize("with_state,use", [(False, (True, False)), (True, (False, True)),
                                            (False, (True, True)), (True, (True, False))])
def test_scan_partial_gradients(TF, with_state, use):
    scan_case(TF, 3, 130, 40, torch.float32, with_state=with_state, use=use)


@pytest.mark.parametrize("mean", [-6.0, 9.0])
def test_scan_gates_near_their_ends(TF, mean):
    scan_case(TF, 2, 1500, 32, torch.float32, mean=mean)


def test_scan_infinite_gates(TF):
    x = randn(1, 6, 8, g=rng(1))
    gate = torch.tensor([9.0, float("inf"), float("inf"), float("-inf"), 0.0, float("inf")],
                        device=DEV).view(1, 6, 1).expand(1, 6, 8)
    y, last = TF.gated_scan(x, gate, torch.ones(1, 8, device=DEV))
    assert torch.equal(y[:, 0], y[:, 1]) and torch.equal(y[:, 1], y[:, 2])  # kept
    assert torch.equal(y[:, 3], x[:, 3])                                      # replaced
    assert torch.equal(y[:, 5], y[:, 4]) and torch.equal(last, y[:, 5])


def test_scan_empty(TF):
    h0 = randn(3, 8, g=rng(1))
    e = torch.zeros(3, 0, 8, device=DEV)
    y, last = TF.gated_scan(e, e, h0)
    assert y.shape == (3, 0, 8) and torch.equal(last, h0)
    z = torch.zeros(0, 4, 8, device=DEV)
    y, last = TF.gated_scan(z, z)
    assert y.shape == (0, 4, 8) and last.shape == (0, 8)


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_step_follows_scan(TF, dtype):
    g = rng(2)
    u = randn(5, 30, 2 * 77, g=g, dtype=dtype)
    x, gate = u.split(77, -1)
    y, last = TF.gated_scan(x, gate)
    state = torch.zeros(5, 77, device=DEV)
    with torch.no_grad():
        for k in range(30):
            yk = TF.gated_scan_step(x[:, k], gate[:, k], state)
            close(yk, y[:, k].double(), rounds=2)
    close(state, last.double())


# ------------------------------------------------------------ differences

def directional(f, leaves, g):
    """(gradient times direction, central difference) of the float64 sum of f's outputs times
    fixed weights."""
    out = f(*leaves)
    outs = out if isinstance(out, tuple) else (out,)
    weights = [randn(*o.shape, g=g) for o in outs]
    grads = torch.autograd.grad(outs, leaves, weights)
    dirs = [randn(*v.shape, g=g) for v in leaves]
    h = 2.0 ** -5

    def value(s):
        with torch.no_grad():
            o = f(*[v + s * d for v, d in zip(leaves, dirs)])
        o = o if isinstance(o, tuple) else (o,)
        return sum((a.double() * b.double()).sum() for a, b in zip(o, weights))

    def slope(s):
        return (value(s) - value(-s)) / (2 * s)

    # Richardson's step removes the h^2 term
    diff = (4 * slope(h / 2) - slope(h)) / 3
    size = sum((a.double() ** 2).sum() for a in grads).sqrt()
    return float(sum((a.double() * b.double()).sum() for a, b in zip(grads, dirs))), float(diff), float(size)


@pytest.mark.parametrize("case", ["layer_norm", "linear", "linear_gelu", "linear_silu", "linear_sigmoid", "scan"])
def test_gradients_against_differences(TF, case):
    g = rng(11)
    if case == "layer_norm":
        leaves = [randn(20, 96, g=g), randn(96, g=g), randn(96, g=g)]
        f = lambda x, w, b: TF.layer_norm(x, w, b)  # noqa: E731
    elif case == "scan":
        leaves = [randn(3, 70, 20, g=g), randn(3, 70, 20, g=g), randn(3, 20, g=g)]
        f = lambda x, a, h: tuple(TF.gated_scan(x, a, h))  # noqa: E731
    else:
        act = case[7:] or None
        leaves = [randn(40, 24, g=g), randn(36, 24, g=g) / 5, randn(36, g=g), randn(40, 36, g=g)]
        f = lambda x, w, b, r: TF.linear(x, w, b, activation=act, residual=r)  # noqa: E731
    got, diff, size = directional(f, [v.requires_grad_(True) for v in leaves], g)
    assert abs(got - diff) <= 2e-3 * size, (got, diff, size)


# ------------------------------------------------------------------ AdamW

def _weights(sizes, dtype, seed=0):
    g = rng(seed)
    ps = [torch.nn.Parameter((0.1 * randn(n, g=g)).to(dtype)) for n in sizes]
    gs = [[(1e-2 * randn(n, g=g)).to(dtype) for n in sizes] for _ in range(4)]
    return ps, gs


def adam_plain(p, gs, lr, b1, b2, eps, wd, dtype):
    """The formula in 64 bits; the weight is rounded to its type at every step."""
    m = v = torch.zeros_like(p, dtype=torch.float64)
    p = p.double()
    for t, gr in enumerate(gs, 1):
        gr = gr.double()
        m = b1 * m + (1 - b1) * gr
        v = b2 * v + (1 - b2) * gr * gr
        p = p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
        p = p.to(dtype).double()
    return p, m, v


SIZES = [1, 255, 256, 257, 5000, 3, 70000, 0, 512]


@pytest.mark.parametrize("dtype", TYPES)
def test_adamw_32_bit(TF, dtype):
    import torchwarp_b200 as tw
    ps, gs = _weights(SIZES, dtype)
    p0 = [p.detach().clone() for p in ps]
    opt = tw.AdamW(ps, lr=3e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    for step in gs:
        for p, gr in zip(ps, step):
            p.grad = gr
        opt.step()
    state = opt.flat_state()
    at = 0
    for k, p in enumerate(ps):
        want, m, v = adam_plain(p0[k], [s[k] for s in gs], 3e-2, 0.8, 0.95, 1e-6, 0.1, dtype)
        # a rounding of the weight to 16 bits may fall to the other side at each of 4 steps
        close(p.detach(), want, rounds=8)
        n = p.numel()
        close(state["exp_avg"][at:at + n], m)
        close(state["exp_avg_sq"][at:at + n], v)
        pad = -(-n // 256) * 256
        assert not state["exp_avg"][at + n:at + pad].any()
        at += pad


def _dither(idx, seed, step):
    mask = 0xFFFFFFFF
    h = (idx ^ ((seed * 0x9E3779B1 + step * 0x85EBCA77) & mask)) & mask
    h = h ^ (h >> 16)
    h = (h * 0x7FEB352D) & mask
    h = h ^ (h >> 15)
    h = (h * 0x846CA68B) & mask
    return h ^ (h >> 16)


@pytest.mark.parametrize("dtype", TYPES)
def test_adamw_8_bit(TF, dtype):
    """Each step against the formula in 64 bits from the states the step began with; the new
    codes lie next to the value on the code's grid."""
    import torchwarp_b200 as tw
    ps, gs = _weights(SIZES, dtype, 1)
    gs[2][4].zero_()
    opt = tw.AdamW(ps, lr=3e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1, state_bits=8, seed=5)
    for t, step in enumerate(gs, 1):
        old = {k: v.clone() for k, v in opt.flat_state().items()}
        before = [p.detach().double() for p in ps]
        for p, gr in zip(ps, step):
            p.grad = gr
        opt.step()
        new = opt.flat_state()
        m0 = (old["exp_avg"].double().view(-1, 256) * old["exp_avg_scale"].double()[:, None]).view(-1)
        r0 = (old["exp_avg_sqrt"].double().view(-1, 256) * old["exp_avg_sqrt_scale"].double()[:, None]).view(-1)
        at = 0
        for k, p in enumerate(ps):
            n = p.numel()
            pad = -(-n // 256) * 256
            gr = torch.nn.functional.pad(step[k].double(), (0, pad - n))
            m = 0.8 * m0[at:at + pad] + (1 - 0.8) * gr
            v = 0.95 * r0[at:at + pad] ** 2 + (1 - 0.95) * gr * gr
            den = (v / (1 - 0.95 ** t)).sqrt()[:n] + 1e-6
            want = before[k] * (1 - 3e-2 * 0.1) - 3e-2 / (1 - 0.8 ** t) * m[:n] / den
            # the update may cancel the weight: the error is relative to what is subtracted
            close(p.detach(), want, floor=F32 * float(before[k].abs().max()) if n else 0.0)
            for name, val in (("exp_avg", m), ("exp_avg_sqrt", v.sqrt())):
                blocks = val.view(-1, 256)
                scale = new[name + "_scale"][at // 256:(at + pad) // 256].double()
                close(scale.float(), blocks.abs().amax(1) / 448 if n else blocks.amax(1))
                y = torch.where(scale[:, None] > 0, blocks.abs() / scale[:, None], blocks * 0)
                ulp = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
                idx = torch.arange(at, at + pad, device=DEV).view(-1, 256)
                h = _dither(idx, 5, t)
                u = (h & 0xFFFF if name == "exp_avg" else h >> 16).double() / 65536
                code = new[name][at:at + pad].double().view(-1, 256)
                q = torch.floor(y / ulp + u) * ulp
                if name == "exp_avg_sqrt":
                    q = torch.where(y > 0, q.clamp(min=2.0 ** -9), q)
                q = q.clamp(max=448) * torch.sign(blocks)
                live = (torch.arange(pad, device=DEV) < n).view(-1, 256)
                off = (code - q)[live]
                # beside a rounding that float32 and float64 see on different sides, the same code
                assert (off.abs() <= (ulp[live] * 1.001)).all()
                assert float((off != 0).double().mean() if n else 0.0) <= 1e-3
            at += pad


def test_adamw_8_bit_moves_slow_averages(TF):
    """With beta2 = 0.999 a step is far below half a code's spacing: the mean still follows."""
    import torchwarp_b200 as tw
    p = torch.nn.Parameter(torch.zeros(256 * 400, device=DEV))
    opt = tw.AdamW([p], lr=0.0, state_bits=8)
    p.grad = torch.ones_like(p)
    for _ in range(300):
        opt.step()
    s = opt.flat_state()
    r = s["exp_avg_sqrt"].double().view(-1, 256) * s["exp_avg_sqrt_scale"].double()[:, None]
    want = math.sqrt(1 - 0.999 ** 300)
    assert abs(float(r.mean()) / want - 1) < 0.05, (float(r.mean()), want)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_many_tensors_views_and_missing_gradients(TF, bits):
    import torchwarp_b200 as tw
    g = rng(3)
    flat = 0.1 * randn(1200 * 9 + 1, g=g)
    ps = [torch.nn.Parameter(flat[1 + 9 * k:1 + 9 * k + 7 + k % 3]) for k in range(1200)]
    p0 = flat.clone()
    opt = tw.AdamW(ps, lr=1e-2, state_bits=bits)
    for k, p in enumerate(ps):
        p.grad = None if k % 5 == 0 else randn(p.numel(), g=g)
    opt.step()
    for k, p in enumerate(ps):
        lo = 1 + 9 * k
        was = p0[lo:lo + p.numel()]
        if k % 5 == 0:
            assert torch.equal(p.detach(), was)
        else:
            close(p.detach(), adam_plain(was, [p.grad], 1e-2, 0.9, 0.999, 1e-8, 1e-2, torch.float32)[0])
    gap = p0.clone()
    for k, p in enumerate(ps):
        gap[1 + 9 * k:1 + 9 * k + p.numel()] = p.detach()
    assert torch.equal(gap, flat)  # nothing written between the tensors


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_checkpoint_graph_and_lr_tensor(TF, bits):
    import torchwarp_b200 as tw

    def run(mode):
        ps, gs = _weights([300, 4096], torch.float32, 2)
        lr = torch.full((), 1e-2, device=DEV)
        opt = tw.AdamW(ps, lr=lr if mode == "graph" else 1e-2, state_bits=bits, seed=3)
        buf = [torch.zeros_like(p) for p in ps]
        for p, b in zip(ps, buf):
            p.grad = b
        graph = None
        for t, step in enumerate(gs):
            for b, gr in zip(buf, step):
                b.copy_(gr)
            if mode == "graph" and t == 1:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.stream(side):
                    with torch.cuda.graph(graph, stream=side):
                        opt.step()
                torch.cuda.current_stream().wait_stream(side)
            if graph is not None:
                graph.replay()
            else:
                opt.step()
            if mode == "load" and t == 1:
                saved = opt.state_dict()
                opt = tw.AdamW(ps, lr=1.0, state_bits=bits)
                opt.load_state_dict(saved)
        torch.cuda.synchronize()
        return [p.detach() for p in ps] + list(opt.flat_state().values())

    plain = run("plain")
    for other in (run("plain"), run("load")):
        for a, b in zip(plain, other):
            assert torch.equal(a.float(), b.float())
    # lr is float32 on the device: 1e-2 differs from the number in its last bits
    for a, b in zip(plain, run("graph")):
        if a.dtype == torch.float32:
            close(b, a.double())


# ---------------------------------------------- streams, compile, modules

def test_operators_run_on_the_current_stream(TF):
    """Inputs made on a side stream, used there at once, read after a wait."""
    side = torch.cuda.Stream()
    g = rng(1)
    x0 = randn(64, 256, g=g)
    w = randn(256, 256, g=g) / 16
    want = linear_plain(ln_plain(x0 * 2, None, None, 1e-5), w, None, None, "silu")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        x = (x0 * 2).requires_grad_(True)
        y = TF.linear(TF.layer_norm(x), w, activation="silu")
        y.sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    close(y.detach(), want, extra=2)
    assert torch.isfinite(x.grad).all()


def test_compile_and_autocast(TF):
    def f(x, w, b, n):
        y = TF.linear(TF.layer_norm(x, n), w, b, activation="gelu")
        v, a = y.split(32, -1)
        out, last = TF.gated_scan(v, a)
        return out.square().sum() + last.sum()

    g = rng(1)
    leaves = [randn(3, 20, 48, g=g), randn(64, 48, g=g) / 7, randn(64, g=g), randn(48, g=g)]
    leaves = [v.requires_grad_(True) for v in leaves]
    want = f(*leaves)
    wg = torch.autograd.grad(want, leaves)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)
    gg = torch.autograd.grad(got, leaves)
    torch.testing.assert_close(got, want)
    for a, b in zip(gg, wg):
        torch.testing.assert_close(a, b)
    with torch.autocast("cuda", torch.bfloat16):
        y = TF.linear(TF.layer_norm(leaves[0], leaves[3]), leaves[1], leaves[2], activation="gelu")
    assert y.dtype == torch.bfloat16
    dx, = torch.autograd.grad(y.float().sum(), leaves[0])
    assert dx.dtype == torch.float32


def test_second_derivative_is_refused(TF):
    x = randn(4, 32, g=rng(1)).requires_grad_(True)
    dx, = torch.autograd.grad(TF.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_encoder_streams_as_it_trains(TF):
    """Frame by frame gives what the whole sequence gives, and the loss falls."""
    import torchwarp_b200 as tw
    torch.manual_seed(0)
    enc = tw.SequenceEncoder(5, 32, layers=2, device=DEV)
    opt = tw.AdamW(enc.parameters(), lr=3e-3, state_bits=8)
    x, y = torch.randn(8, 40, 5, device=DEV), torch.randn(8, 36, 32, device=DEV)
    losses = []
    for _ in range(30):
        opt.zero_grad()
        loss = TF.soft_dtw(enc(x), y, gamma=0.1).mean()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.9 * losses[0], losses
    with torch.no_grad():
        whole = enc(x, lengths=torch.full((8,), 25, device=DEV))
        states = enc.init_state(8)
        for k in range(25):
            got = enc.step(x[:, k], states)
            # the same products through kernels for other row counts
            torch.testing.assert_close(got, whole[:, k], rtol=1e-4, atol=1e-5)
