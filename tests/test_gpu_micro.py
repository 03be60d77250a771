"""The ray-head operators on the GPU against the 64-bit oracle.  Quantised
values are compared bit for bit; sums within the bound of an f32 sum in any
order, (terms + 2) 2^-23 of the sum of magnitudes, plus one rounding to the
result's type."""
import numpy as np
import pytest
import torch

from tests import micro_oracle as O
from vorotracing_amd import micro

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
ACTS = ["none", "relu", "silu", "gelu"]


def _rows(shape, dtype, seed, gpu, special=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-6, 7, (*shape[:-1], 1), generator=g).float())
    if x.numel() and special:
        flat = x.view(-1)
        at = torch.randperm(flat.numel(), generator=g)[:8]
        for i, v in zip(at.tolist(), (0.0, -0.0, float("nan"), float("inf"), -float("inf"), 1e-41, 65504.0, -6e-8)):
            flat[i] = v
        x[..., 0, :] = 0
    return x.to(dtype).to(gpu)


def _within(got, want, allowed, what=""):
    want = O.held(want, got.dtype)
    got = O.f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), (what, "NaN places", int((np.isnan(got) != nan).sum()))
    allowed = np.broadcast_to(allowed, want.shape)
    with np.errstate(invalid="ignore"):
        off = np.where(nan | (got == want), 0.0, np.abs(got - want))
    assert (off <= allowed)[~nan].all(), (what, float(np.nanmax(np.where(nan, 0, off / np.maximum(allowed, 1e-300)))))


SHAPES = [(1, 1), (3, 31), (5, 32), (2, 33), (7, 100), (64, 256), (129, 77), (0, 64), (4, 0), (1, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_and_back(gpu, shape, dtype):
    x = _rows(shape, dtype, 1, gpu, special=True)
    q = micro.quantize_mx4(x)
    codes, scales, v = O.mx4(O.f64(x))
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert tuple(q.shape) == shape
    for to in TYPES:
        with np.errstate(over="ignore"):
            want = torch.from_numpy(v).to(to)
        got = q.dequantize(to).cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_quantize_every_rounding(gpu):
    """Quotients over all of [0, 8), on, beside and between the ties, at the ends of the scale's range."""
    q = np.concatenate([np.arange(0, 8, 1 / 64), [0.25 + 2.0 ** -24, 0.25 - 2.0 ** -26, 5 + 2.0 ** -21, 5 - 2.0 ** -22]])
    rows = []
    for e in (-149, -128, -127, -126, -3, 0, 40, 125):
        for v in q:
            row = np.zeros(32)
            row[0], row[5], row[31] = 4.0, v, -v  # 4 fixes the scale where v is smaller
            with np.errstate(under="ignore"):
                rows.append((row * 2.0 ** float(e)).astype(np.float32))
    x = torch.from_numpy(np.stack(rows)).to(gpu)
    got = micro.quantize_mx4(x)
    codes, scales, _ = O.mx4(O.f64(x))
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.codes.cpu().numpy(), codes)


def test_strided_and_broadcast_rows(gpu):
    base = _rows((40, 200), F16, 2, gpu)
    for x in (base[3:29:2, 7:140], base[:, ::3], base.t(), base[5].expand(6, 200), base.view(4, 10, 200)[:, 2:5, :64],
              base[0]):
        q = micro.quantize_mx4(x)
        want = O.mx4(O.f64(x.contiguous()).reshape(-1, x.shape[-1]))
        assert np.array_equal(q.codes.cpu().numpy().reshape(want[0].shape), want[0])
        assert tuple(q.shape) == tuple(x.shape)
        y, kept = micro.checkpoint_activation(x, "relu")
        c, s, v = O.ckpt8(O.f64(x.contiguous()).reshape(-1, x.shape[-1]))
        assert np.array_equal(kept.codes.cpu().numpy().reshape(c.shape), c) and torch.equal(y, x.clamp(min=0))
        dz = kept.input_grad(x)
        assert torch.equal(dz, torch.where(x > 0, x, torch.zeros_like(x)))


def _weights(out, width, seed, gpu):
    w = micro.quantize_mx4(_rows((out, width), F32, seed, gpu))
    bias = torch.randn(out, generator=torch.Generator().manual_seed(seed)).to(gpu)
    return w, bias


def _linear_want(x, w, bias, relu):
    """(value, sum of magnitudes) in 64 bits."""
    y, s = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, s = y + bias, s + np.abs(bias)
    return (np.where(np.isnan(y), y, np.maximum(y, 0)) if relu else y), s


LINEAR = [(1, 1, 1), (1, 512, 768), (1, 33, 1000), (2, 64, 16), (13, 100, 33), (16, 2048, 64), (17, 256, 256), (31, 31, 31),
          (33, 65, 130), (64, 128, 48), (100, 1000, 7), (130, 256, 256), (257, 333, 520), (300, 64, 300), (1000, 96, 1),
          (2050, 512, 40), (0, 64, 8), (5, 64, 0), (5, 0, 3), (40, 0, 3), (70, 2049, 200), (200, 600, 300), (150, 513, 128),
          (33, 7000, 5)]


@pytest.mark.parametrize("size", LINEAR)
@pytest.mark.parametrize("dtype,to,relu,biased,stored", [
    (F32, F32, False, True, False), (F16, F16, True, True, False), (BF16, BF16, False, False, False),
    (BF16, F32, True, False, True), (F32, BF16, False, True, True)])
def test_linear(gpu, size, dtype, to, relu, biased, stored):
    rows, width, out = size
    x = _rows((rows, width), dtype, 3, gpu)
    w, bias = _weights(out, width, 4, gpu)
    bias = bias if biased else None
    arg = micro.quantize_mx4(x) if stored else x
    got = micro.linear_mx4(arg, w, bias, relu=relu, dtype=to)
    assert got.dtype == to and tuple(got.shape) == (rows, out)
    want, s = _linear_want(O.mx4(O.f64(x))[2], O.f64(w.dequantize()), None if bias is None else O.f64(bias), relu)
    _within(got, want, (width + 2) * 2.0 ** -23 * s + O.rounding(want, to), size)


@pytest.mark.parametrize("size", [(3, 96, 40), (200, 96, 40), (200, 96, 300)])
@pytest.mark.parametrize("stored", [False, True])
def test_linear_keeps_nan_to_its_rows_and_columns(gpu, size, stored):
    rows, width, out = size
    x = _rows((rows, width), F32, 5, gpu)
    x[1, 40] = float("nan")
    x[2, 0] = float("inf")
    wv = _rows((out, width), F32, 6, gpu)
    wv[3, 95] = -float("inf")
    w = micro.quantize_mx4(wv)
    for relu in (False, True):
        got = micro.linear_mx4(micro.quantize_mx4(x) if stored else x, w, relu=relu)
        bad = torch.zeros(rows, out, dtype=torch.bool, device=gpu)
        bad[1:3] = True
        bad[:, 3] = True
        assert torch.equal(got.isnan(), bad)


def _exact_layers(widths, seed, gpu):
    """Layers whose sums are exact in f32: whole weights of at most 6, scales 1."""
    g = torch.Generator().manual_seed(seed)
    layers = []
    for a, b in zip(widths, widths[1:]):
        w = torch.randint(-6, 7, (b, a), generator=g).float()
        w[:, ::32] = 4.0  # each block's scale is 1
        w[w.abs() == 5] = 3.0
        layers.append((micro.quantize_mx4(w.to(gpu)), (torch.randint(-64, 65, (b,), generator=g) / 8).to(gpu)))
    return layers


MLP = [(1, [60, 128, 33]), (13, [60, 128, 128, 33]), (5, [3, 16, 1]), (77, [64, 256, 256, 256, 64]), (129, [27, 33, 75, 10]),
       (300, [256, 256]), (65, [40, 300, 20]), (33, [500, 64, 600, 5]), (0, [8, 8]), (64, [32, 32, 32, 32, 32, 32]),
       (2, [16, 31, 1, 31, 64])]


@pytest.mark.parametrize("rows,widths", MLP)
@pytest.mark.parametrize("dtype,to", [(F32, F32), (F16, F32), (BF16, BF16), (F32, F16)])
def test_mlp(gpu, rows, widths, dtype, to):
    layers = _exact_layers(widths, 7, gpu)
    x = (_rows((rows, widths[0]), F32, 8, gpu) / 64).to(dtype)
    got = micro.mlp_mx4(x, layers, dtype=to)
    h = O.f64(x)
    for i, (w, b) in enumerate(layers):
        h, s = _linear_want(O.mx4(h)[2], O.f64(w.dequantize()), O.f64(b), i + 1 < len(layers))
        if i + 1 < len(layers):  # what goes to 4 bits is the f32 sum itself
            assert np.array_equal(h, h.astype(np.float32)), "the test's sums are to be exact"
    _within(got, h, (layers[-1][0].width + 2) * 2.0 ** -23 * s + O.rounding(h, to), widths)


@pytest.mark.parametrize("rows,widths", [(3000, [40, 70, 33, 9]), (777, [256, 256, 256, 64]), (30, [60, 128, 128, 33])])
def test_mlp_rounds_as_its_layers_do(gpu, rows, widths):
    """Biases of all bits: the sums of one layer's 4-bit products are exact in f32, the bias is their one rounding in
    every form of the product, and so the head's hidden values, scales and results are the layers', bit for bit."""
    g = torch.Generator().manual_seed(34)
    layers = [(micro.quantize_mx4((torch.randn(b, a, generator=g) / a ** 0.5).to(gpu)),
               (0.1 * torch.randn(b, generator=g)).to(gpu)) for a, b in zip(widths, widths[1:])]
    x = torch.randn(rows, widths[0], generator=g).to(gpu)
    h = x
    for i, (w, b) in enumerate(layers):
        q, v = O.mx4(O.f64(h))[2], O.f64(w.dequantize())
        h = micro.linear_mx4(h, w, b, relu=i + 1 < len(layers))
        want = (q @ v.T).astype(np.float32) + O.f64(b).astype(np.float32)
        assert np.array_equal(O.f64(h), np.maximum(want, 0) if i + 1 < len(layers) else want)
    assert torch.equal(micro.mlp_mx4(x, layers), h)


def test_mlp_is_its_layers_in_turn(gpu):
    """More rows than one pass over the workspace, and a NaN row that stays alone."""
    layers = _exact_layers([16, 288, 8], 9, gpu)
    x = _rows((70001, 16), F16, 10, gpu)
    x[69000, 3] = float("nan")
    got = micro.mlp_mx4(x, layers, dtype=F32)
    h = micro.linear_mx4(x, *layers[0], relu=True, dtype=F32)
    want = micro.linear_mx4(h, *layers[1])
    assert torch.equal(got.isnan(), want.isnan()) and bool(got[69000].isnan().all())
    assert torch.equal(got.nan_to_num(), want.nan_to_num()) and int(got.isnan().any(1).sum()) == 1


def test_many_rows_go_round(gpu):
    """More rows than the blocks of the product and of the head take at once."""
    x = _rows((140001, 40), F16, 27, gpu)
    w, bias = _weights(9, 40, 28, gpu)
    for arg in (x, micro.quantize_mx4(x)):
        got = micro.linear_mx4(arg, w, bias, dtype=F32)
        want, s = _linear_want(O.mx4(O.f64(x))[2], O.f64(w.dequantize()), O.f64(bias), False)
        _within(got, want, 42 * 2.0 ** -23 * s + O.rounding(want, F32))
    layers = _exact_layers([40, 70, 33, 9], 29, gpu)
    for dtype in TYPES:
        y = (x.float() / 64).to(dtype)
        got = micro.mlp_mx4(y, layers, dtype=F32)
        h = y
        for i, (weight, b) in enumerate(layers):
            h = micro.linear_mx4(h, weight, b, relu=i < 2, dtype=F32)
        assert torch.equal(got, h)


def test_offsets_past_32_bits(gpu):
    """Tensors of more than 2^32 values: their last rows are those of a call on them alone."""
    x = torch.randn(5_000_000, 1024, device=gpu, dtype=BF16)
    end = x[-100:].clone()
    q, want = micro.quantize_mx4(x), micro.quantize_mx4(end)
    assert torch.equal(q.codes[-100:], want.codes) and torch.equal(q.scales[-100:], want.scales)
    back = q.dequantize(BF16)
    assert torch.equal(back[-100:], want.dequantize(BF16))
    del back
    w, bias = _weights(3, 1024, 33, gpu)
    got = micro.linear_mx4(q, w, bias)  # codes of 2.6 GB
    assert torch.equal(got[-100:], micro.linear_mx4(want, w, bias))
    del q, got
    y, kept = micro.checkpoint_activation(x, "relu")
    want_y, want_kept = micro.checkpoint_activation(end, "relu")
    assert torch.equal(y[-100:], want_y) and torch.equal(kept.codes[-100:], want_kept.codes)
    del y
    dz = kept.input_grad(x)
    assert torch.equal(dz[-100:], want_kept.input_grad(end))
    del dz, x
    dy = torch.zeros(5_000_000, 2, device=gpu, dtype=BF16)
    dy[-64:] = 1
    dw, db = kept.weight_grad(dy)
    last = kept.dequantize(BF16)[-64:].float().clamp(min=0).double()
    assert torch.allclose(dw.double(), last.sum(0).expand(2, -1), rtol=1e-5, atol=1e-5) and db.tolist() == [64.0, 64.0]
    del kept
    x = torch.randn(70_000_000, 1, device=gpu, dtype=F16)
    w, bias = _weights(64, 1, 31, gpu)
    y = micro.linear_mx4(x, w, bias)
    assert torch.equal(y[-100:], micro.linear_mx4(x[-100:], w, bias))
    layers = _exact_layers([1, 32, 64], 32, gpu)
    y = micro.mlp_mx4(x, layers)
    assert torch.equal(y[-100:], micro.mlp_mx4(x[-100:], layers))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_checkpoint_and_input_grad(gpu, shape, dtype, act):
    z = _rows(shape, dtype, 11, gpu, special=True)
    z = z.clamp(-80, 80) if act in ("silu", "gelu") else z  # exp's range: infinities have no slope there
    y, kept = micro.checkpoint_activation(z, act)
    codes, scales, v = O.ckpt8(O.f64(z))
    assert np.array_equal(kept.scales.cpu().numpy(), scales)
    assert np.array_equal(kept.codes.cpu().numpy(), codes)
    zd = O.f64(z)
    _within(y, O.act(zd, act), O.act_error(zd, act) + (O.rounding(O.act(zd, act), dtype) if act in ("silu", "gelu") else 0),
            "y")
    assert y.dtype == dtype
    for to in TYPES:
        assert torch.equal(kept.dequantize(to).cpu().nan_to_num(7.0), torch.from_numpy(v).to(to).nan_to_num(7.0))
    dy = _rows(shape, dtype, 12, gpu)
    dz = kept.input_grad(dy)
    d = O.f64(dy)
    want = d * O.slope(v, act)
    _within(dz, want, np.abs(d) * O.slope_error(v, act) + O.rounding(want, dtype), "dz")


def test_checkpoint_every_rounding(gpu):
    q = np.concatenate([O.E4M3, (O.E4M3[1:] + O.E4M3[:-1]) / 2, [2.0 ** -10, 2.0 ** -11, 2.0 ** -30, 200.0, 248.0, 255.9]])
    q = q[q < 256]
    rows = []
    for e in (-149, -120, -3, 0, 40, 119):
        for v in q:
            row = np.zeros(32)
            row[0], row[5], row[31] = 128.0, v, -v
            with np.errstate(under="ignore"):
                rows.append((row * 2.0 ** float(e)).astype(np.float32))
    x = torch.from_numpy(np.stack(rows)).to(gpu)
    kept = micro.checkpoint_activation(x, "none")[1]
    codes, scales, _ = O.ckpt8(O.f64(x))
    assert np.array_equal(kept.scales.cpu().numpy(), scales)
    assert np.array_equal(kept.codes.cpu().numpy(), codes)


WEIGHTS = [(1, 1, 1), (5, 33, 7), (64, 32, 16), (100, 77, 130), (1000, 128, 128), (777, 200, 333), (3000, 256, 256),
           (4099, 31, 1), (2500, 1, 65), (0, 40, 8), (20, 0, 5), (20, 5, 0), (9000, 130, 5)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", WEIGHTS)
def test_weight_grad(gpu, size, dtype, act):
    rows, width, out = size
    z = (_rows((rows, width), F32, 13, gpu) / 8).clamp(-60, 60)
    kept = micro.checkpoint_activation(z, act)[1]
    dy = _rows((rows, out), dtype, 14, gpu)
    dw, db = kept.weight_grad(dy)
    assert dw.dtype == db.dtype == F32 and tuple(dw.shape) == (out, width) and tuple(db.shape) == (out,)
    d, v = O.f64(dy), O.ckpt8(O.f64(z))[2]
    a, ad = O.act(v, act), np.abs(d)
    # a product's factors are within act_error and, in parts of 8 bits, 2^-22 of themselves
    _within(dw, d.T @ a, (rows + 4) * 2.0 ** -23 * (ad.T @ np.abs(a)) + ad.T @ O.act_error(v, act)
            + 2.0 ** -22 * (ad.T @ np.abs(a)) + 1e-36, "dw")
    _within(db, d.sum(0), (rows + 2) * 2.0 ** -23 * ad.sum(0), "db")
    again = kept.weight_grad(dy)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1])


def test_weight_grad_of_tiny_activations(gpu):
    """Blocks under the smallest scale: values whose bf16 is subnormal (multiples of 2^-133 at least are exact)."""
    z = (_rows((64, 40), F32, 26, gpu).sign() * 2.0 ** -127).contiguous()
    z[:, ::3] *= 0.375
    for act in ("none", "relu"):
        kept = micro.checkpoint_activation(z, act)[1]
        assert int(kept.scales.max()) == 0
        dy = torch.full((64, 8), 2.0 ** 100, device=gpu).bfloat16()
        dw, _ = kept.weight_grad(dy)
        a = O.act(O.ckpt8(O.f64(z))[2], act)
        assert np.array_equal(O.f64(dw), np.broadcast_to(2.0 ** 100 * a.sum(0), (8, 40)))


def test_weight_grad_against_differences(gpu):
    """The loss sum(dy * (act(z^) W^T + b)) is linear in W and b: its differences, in 64 bits, are the gradients."""
    z = _rows((50, 40), F32, 15, gpu) / 8
    kept = micro.checkpoint_activation(z, "gelu")[1]
    dy = _rows((50, 6), F32, 16, gpu) / 8
    dw, db = kept.weight_grad(dy)
    a, d = O.act(O.f64(kept.dequantize()), "gelu"), O.f64(dy)
    rng = np.random.default_rng(0)
    w, b = rng.normal(size=(6, 40)), rng.normal(size=6)
    loss = lambda w, b: (d * (a @ w.T + b)).sum()  # noqa: E731
    for _ in range(5):
        e, f = rng.normal(size=w.shape), rng.normal(size=b.shape)
        diff = (loss(w + e, b + f) - loss(w - e, b - f)) / 2
        got = (O.f64(dw) * e).sum() + (O.f64(db) * f).sum()
        scale = (np.abs(d).T @ np.abs(a) * np.abs(e)).sum() + (np.abs(d).sum(0) * np.abs(f)).sum()
        assert abs(diff - got) <= 64 * 2.0 ** -21 * scale


def test_input_grad_against_differences(gpu):
    """Differences of the operator's own values at the points the checkpoint holds."""
    for act in ("silu", "gelu"):
        z = torch.linspace(-6, 6, 512, device=gpu).view(8, 64)
        kept = micro.checkpoint_activation(z, act)[1]
        v = kept.dequantize(F32)
        h = 2.0 ** -6
        up, down = (micro.checkpoint_activation(v + s * h, act)[0].double() for s in (1, -1))
        dz = kept.input_grad(torch.ones_like(z)).double()
        # third derivative below 2: h^2 / 3; values up to 6 rounded to 2^-21 of themselves over 2 h
        assert float(((up - down) / (2 * h) - dz).abs().max()) < h * h / 3 * 2 + 6 * 2.0 ** -21 / h


def test_weight_grad_nan_stays_in_its_row_and_column(gpu):
    z = _rows((600, 70), F32, 17, gpu)
    z[5, 40] = float("nan")
    dy = _rows((600, 50), F32, 18, gpu)
    dy[7, 9] = float("inf")
    kept = micro.checkpoint_activation(z, "relu")[1]
    dw, db = kept.weight_grad(dy)
    assert bool(dw[:, 40].isnan().all())
    rest = dw.clone()
    rest[:, 40] = 0
    rest[9] = 0
    assert bool(rest.isfinite().all())
    assert bool((~dw[9].isfinite()).any()) and db[9] == float("inf") and int((~db.isfinite()).sum()) == 1


def test_streams_and_shared_buffers(gpu):
    """Calls on a stream of their own, their inputs made on it, give the same results."""
    x = _rows((500, 200), BF16, 19, gpu)
    w, bias = _weights(96, 200, 20, gpu)
    want = micro.linear_mx4(x, w, bias)
    layers = _exact_layers([200, 300, 40], 21, gpu)
    want_mlp = micro.mlp_mx4(x, layers)
    kept = micro.checkpoint_activation(x, "silu")[1]
    want_dw = kept.weight_grad(x)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            y = x.clone()
            got, mlp = micro.linear_mx4(y, w, bias), micro.mlp_mx4(y, layers)
            dw = micro.checkpoint_activation(y, "silu")[1].weight_grad(y)[0]
            del y
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(mlp, want_mlp) and torch.equal(dw, want_dw)


def test_replayed_from_a_graph(gpu):
    x = _rows((300, 200), F32, 22, gpu)
    w, bias = _weights(96, 200, 23, gpu)
    layers = _exact_layers([200, 64, 40], 24, gpu)

    def step():
        y, kept = micro.checkpoint_activation(x, "relu")
        return (micro.linear_mx4(x, w, bias), micro.mlp_mx4(x, layers), y, kept.input_grad(x), *kept.weight_grad(x),
                micro.quantize_mx4(x).dequantize())

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        x.copy_(_rows((300, 200), F32, 30 + i, gpu))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_refusals(gpu):
    x = torch.zeros(4, 64, device=gpu)
    w, bias = _weights(8, 64, 25, gpu)
    with pytest.raises(ValueError, match="64 values with weights of"):
        micro.linear_mx4(x, _weights(8, 65, 25, gpu)[0])
    with pytest.raises(ValueError, match="float32 tensor of 8"):
        micro.linear_mx4(x, w, bias[:7])
    with pytest.raises(ValueError, match="float32 tensor of 8"):
        micro.linear_mx4(x, w, bias.half())
    with pytest.raises(ValueError, match="weights are an Mx4"):
        micro.linear_mx4(x, x)
    with pytest.raises(ValueError, match="got torch.float64"):
        micro.linear_mx4(x, w, dtype=torch.float64)
    with pytest.raises(ValueError, match="records no gradient"):
        micro.linear_mx4(x.clone().requires_grad_(), w)
    with pytest.raises(ValueError, match="records no gradient"):
        micro.mlp_mx4(x, [(w, bias.clone().requires_grad_())])
    with torch.no_grad():
        micro.linear_mx4(x.clone().requires_grad_(), w, bias.clone().requires_grad_())
    with pytest.raises(ValueError, match="1 to 16 layers"):
        micro.mlp_mx4(x, [])
    with pytest.raises(ValueError, match="8 values with weights of"):
        micro.mlp_mx4(x, [(w, bias), (w, bias)])
    with pytest.raises(ValueError, match="expected rows of 32"):
        micro.Mx4(w.codes[:, :16], w.scales, 64)
    with pytest.raises(ValueError, match="contiguous"):
        micro.Mx4(w.codes.t().contiguous().t(), w.scales, 64)
    kept = micro.checkpoint_activation(x, "silu")[1]
    with pytest.raises(ValueError, match="for activations of"):
        kept.input_grad(x[:3])
    with pytest.raises(ValueError, match="for activations of"):
        kept.weight_grad(x[:3])
    with pytest.raises(ValueError, match="none of none, relu, silu, gelu"):
        micro.checkpoint_activation(x, "tanh")
    with pytest.raises(ValueError, match="got a scalar"):
        micro.quantize_mx4(torch.zeros((), device=gpu))
