"""The encoder operators in a program: a training step captured as a CUDA graph, the same bits at
every run, and tensors of more than 2^31 elements (B200).

The comparisons of the large tensors are with the same operator on a slice that holds their last
rows, which the other tests compare with 64-bit forms; rows are independent, so the bits are equal
where the slice takes the same kernels.
"""

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


def _program(tw, bits):
    torch.manual_seed(3)
    enc = tw.SequenceEncoder(6, 32, layers=2, device=DEV)
    opt = tw.AdamW(enc.parameters(), lr=2e-3, state_bits=bits, seed=1)
    crit = tw.SoftDTW(gamma=0.5)

    def step(x, y):
        loss = crit(enc(x), y).mean()
        opt.zero_grad(set_to_none=False)
        loss.backward()
        opt.step()
        return loss

    return enc, step


def _batches():
    g = torch.Generator(device=DEV).manual_seed(4)
    return [(torch.randn(9, 50, 6, device=DEV, generator=g),
             torch.randn(9, 44, 32, device=DEV, generator=g)) for _ in range(6)]


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_step_gives_the_bits_of_the_eager_one(tw, bits):
    batches = _batches()
    enc, step = _program(tw, bits)
    eager = [step(x, y).item() for x, y in batches]
    want = [p.detach().clone() for p in enc.parameters()]

    enc, step = _program(tw, bits)
    again = [step(x, y).item() for x, y in batches]
    assert again == eager  # one result for one program
    for p, w in zip(enc.parameters(), want):
        assert torch.equal(p, w)

    enc, step = _program(tw, bits)
    sx, sy = (torch.empty_like(t) for t in batches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, y in batches[:3]:
            sx.copy_(x)
            sy.copy_(y)
            step(sx, sy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(sx, sy)
    replayed = []
    for x, y in batches[3:]:
        sx.copy_(x)
        sy.copy_(y)
        graph.replay()
        replayed.append(loss.item())
    assert replayed == eager[3:]
    for p, w in zip(enc.parameters(), want):
        assert torch.equal(p, w)
    assert tw._native.lib().tw_device_error() == 0


def test_zero_sized_parameters_alone(tw):
    p = torch.nn.Parameter(torch.zeros(0, 4, device=DEV))
    p.grad = torch.zeros_like(p)
    tw.AdamW([p]).step()
    torch.cuda.synchronize()


ROWS = 2 ** 21 + 77  # of 1024: over 2^31 elements


def _large(fill=1.0):
    x = torch.empty(ROWS, 1024, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(5)
    x.normal_(generator=g).mul_(fill)
    return x


def test_layer_norm_past_32_bits(tw):
    TF = tw.functional
    x, dy = _large().requires_grad_(True), _large(0.5)
    w = torch.rand(1024, device=DEV).bfloat16()
    y = TF.layer_norm(x, w)
    dx, = torch.autograd.grad(y, x, dy)
    xs = x.detach()[-64:].clone().requires_grad_(True)
    ys = TF.layer_norm(xs, w)
    dxs, = torch.autograd.grad(ys, xs, dy[-64:].contiguous())
    assert torch.equal(y[-64:], ys) and torch.equal(dx[-64:], dxs)


def test_linear_past_32_bits(tw):
    TF = tw.functional
    x, w = _large(), (torch.randn(1024, 1024, device=DEV) / 32).bfloat16()
    r = _large(0.5)
    y = TF.linear(x, w, activation="gelu", residual=r)
    # the last rows at the place they have in their tiles, by the same kernel
    n = 256 * 200 + ROWS % 256
    ys = TF.linear(x[-n:], w, activation="gelu", residual=r[-n:])
    assert torch.equal(y[-n:], ys)
    rows = slice(0, ROWS, 65537)
    want = torch.nn.functional.gelu(x[rows].double() @ w.double().t()) + r[rows].double()
    err = float((y[rows].double() - want).norm() / want.norm())
    assert err <= 2.0 ** -8, err


def test_gated_scan_past_32_bits(tw):
    TF = tw.functional
    T = 700_001  # x 3 x 1024
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.empty(3, T, 1024, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    gate = torch.empty_like(x).normal_(generator=g)  # a state lasts a few frames
    x.requires_grad_(True)
    y, last = TF.gated_scan(x, gate)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    # the last 300 frames alone: what came before has decayed below a rounding
    xs = x.detach()[:, -300:].clone().requires_grad_(True)
    ys, lasts = TF.gated_scan(xs, gate[:, -300:].contiguous())
    dxs, = torch.autograd.grad(ys, xs, torch.ones_like(ys))
    torch.testing.assert_close(last, lasts, rtol=1e-5, atol=1e-6)
    for a, b in ((y[:, -100:], ys[:, -100:]), (dx[:, -100:], dxs[:, -100:])):
        torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-6)


def test_linear_bias_gradient_of_nearly_2_to_31_rows(tw):
    """The last of the blocks of rows ends past 2^31: its rows count."""
    import torchwarp_b200._native as nat
    rows, n = 2 ** 31 - 1000, 8
    dy = torch.zeros(rows, n, device=DEV, dtype=torch.bfloat16)
    dy[-5:] = 3
    lib = nat.lib()
    size = lib.tw_linear_workspace_bytes(rows, n, 8, 2, 0, 1, 0)
    ws = torch.empty(size, device=DEV, dtype=torch.uint8)
    db = torch.empty(n, device=DEV, dtype=torch.bfloat16)
    x = torch.empty(8, device=DEV, dtype=torch.bfloat16)  # not read: only db is asked for
    status = lib.tw_linear_backward_bf16(dy.data_ptr(), n, x.data_ptr(), 8, x.data_ptr(), 8, None,
                                         rows, n, 8, 0, None, None, db.data_ptr(), ws.data_ptr(),
                                         size, torch.cuda.current_stream().cuda_stream)
    assert status == 0 and (db == 15).all()
