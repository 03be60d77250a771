"""The ray head on the GPU: its layers against the formulas in 64 bits, what it
keeps between the passes, training through the tracer, and serving."""
import numpy as np
import pytest
import torch

from tests import helpers as H
from tests import micro_oracle as O
from vorotracing_amd import camera, head, micro
from vorotracing_amd.infer import VoroTracingInfer
from vorotracing_amd.model import VoroTracing

pytestmark = pytest.mark.gpu

BITS = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", list(BITS))
@pytest.mark.parametrize("lead,width,out", [((7,), 33, 5), ((3, 40), 64, 48), ((300,), 31, 1)])
def test_activated_linear_against_the_formulas(gpu, lead, width, out, dtype, act):
    g = torch.Generator().manual_seed(1)
    z = torch.randn((*lead, width), generator=g).to(dtype).to(gpu).requires_grad_()
    w = (torch.randn((out, width), generator=g) / width ** 0.5).to(gpu).requires_grad_()
    b = torch.randn(out, generator=g).to(gpu).requires_grad_()
    dy = torch.randn((*lead, out), generator=g).to(dtype).to(gpu)
    y = head.activated_linear(z, w, b, act)
    assert y.dtype == dtype and tuple(y.shape) == (*lead, out)
    y.backward(dy)
    # operands rounded to the type (2^-p each), an f32 sum in any order, the result rounded to the type
    u, f = 2.0 ** -BITS[dtype], 2.0 ** -23
    zd, wd, bd, d = O.f64(z).reshape(-1, width), O.f64(w), O.f64(b), O.f64(dy).reshape(-1, out)
    a = O.act(zd, act)
    want, s = a @ wd.T + bd, np.abs(a) @ np.abs(wd).T + np.abs(bd)
    allowed = (2.1 * u + (width + 2) * f) * s + O.act_error(zd, act) @ np.abs(wd).T + u * np.abs(want)
    assert (np.abs(O.f64(y).reshape(-1, out) - want) <= allowed).all()
    v = O.ckpt8(zd)[2]  # the backward pass is that of the values kept
    t, ts = d @ wd, np.abs(d) @ np.abs(wd)
    want = t * O.slope(v, act)
    allowed = ((1.1 * u + (out + 2) * f) * ts + u * np.abs(t)) * 1.2 + ts * O.slope_error(v, act) + u * np.abs(want)
    assert (np.abs(O.f64(z.grad).reshape(-1, width) - want) <= allowed).all()
    av, rows = O.act(v, act), d.shape[0]
    s = np.abs(d).T @ np.abs(av)
    assert (np.abs(O.f64(w.grad) - d.T @ av) <= ((rows + 4) * f + 2 * f) * s + np.abs(d).T @ O.act_error(v, act)).all()
    assert (np.abs(O.f64(b.grad) - d.sum(0)) <= (rows + 2) * f * np.abs(d).sum(0)).all()


def test_four_bit_layer_is_the_served_product(gpu):
    g = torch.Generator().manual_seed(2)
    z = torch.randn(50, 70, generator=g).to(gpu).requires_grad_()
    w = torch.randn(9, 70, generator=g).to(gpu).requires_grad_()
    b = torch.randn(9, generator=g).to(gpu).requires_grad_()
    dy = torch.randn(50, 9, generator=g).to(gpu)
    y = head.activated_linear(z, w, b, "relu", four_bit=True)
    wq = micro.quantize_mx4(w.detach())
    assert torch.equal(y, micro.linear_mx4(z.detach().clamp(min=0), wq, b.detach()))
    y.backward(dy)
    d, wd = O.f64(dy), O.mx4(O.f64(w))[2]
    kept = micro.checkpoint_activation(z.detach(), "relu")[1]
    want = d @ wd * (O.f64(z) > 0)
    assert (np.abs(O.f64(z.grad) - want) <= 11 * 2.0 ** -23 * (np.abs(d) @ np.abs(wd))).all()
    dw, db = kept.weight_grad(dy)
    assert torch.equal(w.grad, dw) and torch.equal(b.grad, db)


def test_no_gradient_that_is_not_asked_for(gpu):
    z = torch.randn(20, 16, device=gpu)
    w = torch.randn(4, 16, device=gpu, requires_grad=True)
    y = head.activated_linear(z, w)
    y.sum().backward()
    assert z.grad is None and w.grad is not None
    with torch.no_grad():
        assert not head.activated_linear(z, w).requires_grad


def test_a_hidden_value_costs_a_byte_between_the_passes(gpu):
    net = head.RayHead([32, 256, 256, 8], device=gpu)
    x = torch.randn(4096, 32, device=gpu)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        net(x)
    params = {p.data_ptr() for p in net.parameters()}
    rows = [t for t in kept if t.data_ptr() not in params and t.shape[0] == 4096]
    values = 4096 * (32 + 256 + 256)
    assert sum(t.numel() * t.element_size() for t in rows) == values + values // 32


def test_trains_with_the_scene_and_serves(gpu):
    s = H.small_random(900, seed=11, R=4)
    rays = H.to_dev(camera.pinhole_rays(40, 32, eye=(0.2, -3.4, 0.3)), gpu)
    model = VoroTracing.from_scene(s, device=gpu)
    torch.manual_seed(3)
    with torch.no_grad():
        rgba = model(rays)[0]
        target = rgba[..., :3] * (0.5 + 0.5 * torch.nn.functional.normalize(rays[..., 3:], dim=-1) ** 2)
    x = head.ray_inputs(rgba, rays)
    assert tuple(x.shape) == (32, 40, 31)
    net = head.RayHead([31, 64, 64, 3], dtype=torch.float32, device=gpu)
    opt = torch.optim.Adam([*net.parameters(), model.att_diffuse], lr=2e-3)
    losses, served = [], []

    def serve_loss():
        image = VoroTracingInfer(model).render(rays)
        out = head.RayHeadInfer(net)(head.ray_inputs(image.float(), rays))
        return float((out - target).square().mean())

    for step in range(120):
        if step == 60:
            net.four_bit = True
            served.append(serve_loss())
        opt.zero_grad()
        loss = (net(head.ray_inputs(model(rays)[0], rays)).float() - target).square().mean()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    served.append(serve_loss())
    assert float(model.att_diffuse.grad.abs().sum()) > 0
    assert losses[59] < 0.1 * losses[0]
    assert served[1] < served[0]  # the steps in 4 bits are for the served head
    serve = head.RayHeadInfer(net)
    for (w, b), layer in zip(serve.layers, net.layers):
        codes, scales, _ = O.mx4(O.f64(layer.weight))
        assert np.array_equal(w.codes.cpu().numpy(), codes) and np.array_equal(w.scales.cpu().numpy(), scales)
        assert torch.equal(b, layer.bias)
    x = head.ray_inputs(rgba, rays)
    out = serve(x)
    assert out.dtype == torch.float32 and tuple(out.shape) == (32, 40, 3)
    # the same products as in training, bias first or last: f32 sums apart by their order, which turns a hidden value
    # at a tie to its other neighbour in few rows
    with torch.no_grad():
        apart = (out - net(x)).abs().amax(-1)
    assert float((apart > 1e-5).float().mean()) < 0.01


def test_refusals(gpu):
    with pytest.raises(ValueError, match="two widths"):
        head.RayHead([4], device=gpu)
    with pytest.raises(ValueError, match="none of none, relu"):
        head.RayHead([4, 4], "tanh", device=gpu)
    with pytest.raises(ValueError, match="16 values with weights of"):
        head.activated_linear(torch.zeros(3, 16, device=gpu), torch.zeros(4, 15, device=gpu))
    with pytest.raises(ValueError, match="runs ReLU between"):
        head.RayHeadInfer(head.RayHead([4, 4, 4], "silu", device=gpu))
    with pytest.raises(ValueError, match="for activations of"):
        micro.checkpoint_activation(torch.zeros(3, 4, device=gpu), "none")[1].weight_grad(torch.zeros(2, 4, device=gpu))
