"""GPU: layer normalisation, Newton-Schulz orthogonalisation and the Muon update against plain implementations in 64 bits.

Tolerances come from the rounding model of the arithmetic, not from runs.  u = 2^-24 is half a step of fp32, a sum of n terms
in a tree or in strided chains is off by at most (its depth) u times the sum of magnitudes; a result rounded to a type T is
off by finfo(T).eps / 2 relative to it (fp16 also by half its smallest step, 2^-25)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
IDS = {F32: "fp32", F16: "fp16", BF16: "bf16"}


def rounded(v, dtype):
    """Half a step of `dtype` at the 64-bit values v."""
    return v.abs() * (torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == F16 else 0.0)


def check(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %g with %g allowed" % (
        what, bad.sum(), bad.numel(), (got - want).abs().max(), (tol if torch.is_tensor(tol) else torch.tensor(tol)).max())


# ---- layer normalisation ---------------------------------------------------------------------------------------------------

def norm_reference(x, w, b, eps, dy=None, dtype=F32, wdtype=F32):
    """(value, tolerance) of y, dx, dw, db in 64 bits."""
    x = x.double()
    rows, n = x.shape
    one = torch.ones(n, dtype=torch.float64, device=x.device)
    w64, b64 = one if w is None else w.double(), 0 * one if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * w64 + b64
    depth = 16 + n / 64                        # of a row's sums: a chain per thread and a tree over a workgroup
    k = depth + 8
    spread = x.abs().mean(1, keepdim=True) * rstd   # the mean's own error, in units of xh: k u mean|x| rstd
    # the variance: relative error from its own sum, from the centred values' rounding and from the mean's error squared
    e_rstd = k * U * (1 + 0 * rstd) + 0.5 * (k * U * spread).square() + U * spread * xh.abs().mean(1, keepdim=True)
    e_xh = k * U * spread + (4 * U + e_rstd) * xh.abs()
    out = [(y, e_xh * w64.abs() + 4 * U * (xh * w64).abs() + 2 * U * y.abs() + rounded(y, dtype))]
    if dy is None:
        return out
    dy = dy.double()
    h = dy * w64
    mh, mx = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    dx = rstd * (h - mh - xh * mx)
    e_mh = k * U * h.abs().mean(1, keepdim=True)
    e_mx = k * U * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * e_xh).mean(1, keepdim=True)
    e_dx = rstd * (4 * U * (h.abs() + mh.abs() + (xh * mx).abs()) + e_mh + xh.abs() * e_mx + e_xh * mx.abs()) + (4 * U + e_rstd) * dx.abs()
    out.append((dx, e_dx + rounded(dx, dtype)))
    deep = 64 + min(rows, 512) + rows / 64      # of a column's sums: chains over rows, then over chunks
    dw, db = (dy * xh).sum(0), dy.sum(0)
    out.append((dw, deep * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0) + rounded(dw, wdtype)))
    out.append((db, deep * U * dy.abs().sum(0) + rounded(db, wdtype)))
    return out


def norm_inputs(rows, cols, dtype, wdtype, seed=0, pad=0, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    def wide():
        buf = torch.randn(rows * (cols + pad) + offset, generator=g, device=DEV)
        return buf.to(dtype)[offset:].view(rows, cols + pad)[:, :cols]
    x, dy = wide() * 2 + torch.randn(rows, 1, generator=g, device=DEV).to(dtype), wide()
    if pad or offset:                          # (arithmetic above makes x contiguous: keep the strides)
        keep = wide()
        keep.copy_(x)
        x = keep
    w = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(wdtype)
    b = torch.randn(cols, generator=g, device=DEV).to(wdtype)
    return x, w, b, dy


def norm_both(x, w, b, dy, eps=1e-5):
    from gan_flow_amd.lib.layers import layer_norm
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    return [y.detach()] + list(grads)


SHAPES = [(1, 1), (1, 7), (4, 2), (3, 64), (64, 3), (5, 100), (300, 257), (2, 1000), (17, 1024), (9, 2048), (7, 4097), (2, 8200), (1, 40000),
          (2049, 16), (700, 512)]


@pytest.mark.parametrize("dtype, wdtype", [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)],
                         ids=lambda t: IDS[t])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_layer_norm_and_its_gradients(rows, cols, dtype, wdtype):
    x, w, b, dy = norm_inputs(rows, cols, dtype, wdtype)
    for name, got, (want, tol) in zip(("y", "dx", "dw", "db"), norm_both(x, w, b, dy), norm_reference(x, w, b, 1e-5, dy, dtype, wdtype)):
        assert got.dtype == (dtype if name in ("y", "dx") else wdtype)
        check(got, want, tol, name)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: IDS[t])
@pytest.mark.parametrize("pad, offset", [(1, 0), (0, 1), (24, 0), (3, 5), (8, 8), (64, 2)])
@pytest.mark.parametrize("rows, cols", [(33, 72), (6, 1001), (4, 2560)])
def test_layer_norm_of_strided_and_unaligned_rows(rows, cols, pad, offset, dtype):
    x, w, b, dy = norm_inputs(rows, cols, dtype, dtype, 1, pad, offset)
    assert rows == 1 or x.stride(0) == cols + pad
    for name, got, (want, tol) in zip(("y", "dx", "dw", "db"), norm_both(x, w, b, dy), norm_reference(x, w, b, 1e-5, dy, dtype, dtype)):
        check(got, want, tol, name)


@pytest.mark.parametrize("has_w, has_b", [(True, False), (False, True), (False, False)])
def test_layer_norm_without_weight_or_bias(has_w, has_b):
    x, w, b, dy = norm_inputs(50, 130, BF16, F32, 2)
    w, b = w if has_w else None, b if has_b else None
    got = norm_both(x, w, b, dy)
    want = norm_reference(x, w, b, 1e-5, dy, BF16, F32)
    picked = [want[0], want[1]] + ([want[2]] if has_w else []) + ([want[3]] if has_b else [])
    for g, (v, tol) in zip(got, picked):
        check(g, v, tol, "output")
    assert len(got) == len(picked)


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("rows, cols", [(40, 200), (40, 3001)])
def test_layer_norm_gradients_one_by_one(wanted, rows, cols):
    from gan_flow_amd import _native as nat
    x, w, b, dy = norm_inputs(rows, cols, F32, F32, 3)
    _, mean, rstd = nat.layer_norm_fwd(x, w, b)
    got = nat.layer_norm_bwd(dy, x, w, mean, rstd, wanted)
    for g, want, (v, tol) in zip(got, wanted, norm_reference(x, w, b, 1e-5, dy)[1:]):
        assert (g is not None) == bool(want)
        if want:
            check(g, v, tol, "gradient")


def test_layer_norm_far_from_zero_and_of_constant_rows():
    x, w, b, dy = norm_inputs(20, 300, F32, F32, 4)
    x[:5] += 1e4                       # far from zero: a variance from moments would lose everything
    x[5:8] = 7.25                      # constant rows: variance 0
    x[8] = 0
    for got, (want, tol) in zip(norm_both(x, w, b, dy), norm_reference(x, w, b, 1e-5, dy)):
        check(got, want, tol, "output")


@pytest.mark.parametrize("cols", [48, 1500, 9000])
def test_layer_norm_keeps_rows_apart(cols):
    from gan_flow_amd.lib.layers import layer_norm
    x, w, b, _ = norm_inputs(6, cols, F32, F32, 5)
    clean = layer_norm(x, w, b)
    x[1, 0], x[3, cols - 1], x[4, 5] = float("nan"), float("inf"), float("-inf")
    y = layer_norm(x, w, b)
    assert torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])
    assert y[[1, 3, 4]].isnan().all()


def test_layer_norm_of_nothing_and_of_many_axes():
    from gan_flow_amd.lib.layers import LayerNorm, layer_norm
    x = torch.randn(0, 12, device=DEV, requires_grad=True)
    w = torch.randn(12, device=DEV, requires_grad=True)
    y = layer_norm(x, w, None)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 12) and gx.shape == (0, 12) and gw.eq(0).all()
    assert layer_norm(torch.randn(3, 0, 8, device=DEV)).shape == (3, 0, 8)
    x, w, b, _ = norm_inputs(24, 40, F32, F32, 6)
    m = LayerNorm(40).to(DEV)
    with torch.no_grad():
        m.weight.copy_(w), m.bias.copy_(b)
    assert torch.equal(m(x.view(2, 3, 4, 40)).reshape(24, 40), layer_norm(x, w, b))
    assert torch.equal(layer_norm(x.t().contiguous().t(), w, b), layer_norm(x, w, b))       # columns contiguous: copied
    assert torch.equal(layer_norm(x[0], w, b), layer_norm(x[:1], w, b)[0])


def test_layer_norm_of_broadcast_gradients_and_rows():
    from gan_flow_amd.lib.layers import layer_norm
    x, w, b, dy = norm_inputs(31, 65, F32, F32, 7)
    lx = x.clone().requires_grad_()
    y = layer_norm(lx, w, b)
    row = dy[:1].expand(31, 65)                                     # row stride 0
    for g in (row, dy[:, :1].expand(31, 65), torch.ones((), device=DEV).expand(31, 65)):
        (got,) = torch.autograd.grad(y, lx, g, retain_graph=True)
        want, tol = norm_reference(x, w, b, 1e-5, g)[1]
        check(got, want, tol, "dx")
    shared = x[:1].expand(31, 65)
    assert torch.equal(layer_norm(shared, w, b), layer_norm(x[:1], w, b).expand(31, 65))


def test_layer_norm_gradient_against_differences():
    """(L(x + h v) - L(x - h v)) / 2 h along a direction: off by h^2 / 6 of the third derivative (bounded from a 64-bit
    evaluation at 2 h) and by the two values' rounding over h."""
    from gan_flow_amd.lib.layers import layer_norm
    x, w, b, dy = norm_inputs(4, 96, F32, F32, 8)
    grads = norm_both(x, w, b, dy)[1:]
    g = torch.Generator(device=DEV).manual_seed(9)
    for i in range(3):
        args = [x, w, b]
        v = torch.randn(args[i].shape, generator=g, device=DEV)
        h = 2.0 ** -6

        def loss(f, s, dt):
            moved = [t.to(dt) for t in args]
            moved[i] = moved[i] + s * v.to(dt)
            return (f(*moved).double() * dy.double()).sum()

        exact = lambda xx, ww, bb: norm_reference(xx, ww, bb, 1e-5)[0][0]  # noqa: E731
        central = lambda f, s, dt: ((loss(f, s, dt) - loss(f, -s, dt)) / (2 * s)).item()  # noqa: E731
        along = (grads[i].double() * v.double()).sum().item()
        truncation = abs(central(exact, 2 * h, torch.float64) - central(exact, h, torch.float64))
        tol_y = norm_reference(x, w, b, 1e-5)[0][1] * 2
        rounding = ((tol_y + U * 8) * dy.double().abs()).sum().item() / h
        assert abs(central(layer_norm, h, F32) - along) <= truncation + rounding + 1e-5 * abs(along)


def test_layer_norm_is_differentiable_once_and_deterministic():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.layers import layer_norm
    x, w, b, dy = norm_inputs(4097, 320, BF16, F32, 10)
    first = norm_both(x, w, b, dy)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, norm_both(x, w, b, dy)))
    lx = x[:8].float().requires_grad_()
    (gx,) = torch.autograd.grad(layer_norm(lx, w, b).square().sum(), lx, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    with pytest.raises(CnfError):
        layer_norm(x, w[:-1], b)
    with pytest.raises(CnfError):
        layer_norm(x, w, b.to(BF16))
    with pytest.raises(CnfError):
        layer_norm(x, w.to(F16), None)
    with pytest.raises(CnfError):
        layer_norm(x.double(), None, None)
    with pytest.raises(CnfError):
        layer_norm(x, w.cpu(), b)
    with pytest.raises(CnfError):
        layer_norm(x[:, :0], None, None)


def test_layer_norm_on_another_stream_and_in_a_graph():
    from gan_flow_amd import _native as nat
    x, w, b, dy = norm_inputs(130, 200, F32, F32, 11)
    want = norm_both(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_both(x, w, b, dy)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    xs, dys = x.clone(), dy.clone()

    def both():
        y, mean, rstd = nat.layer_norm_fwd(xs, w, b)
        return (y,) + nat.layer_norm_bwd(dys, xs, w, mean, rstd)

    both()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(both())
    for seed in range(3):
        x2, _, _, dy2 = norm_inputs(130, 200, F32, F32, 20 + seed)
        want = norm_both(x2, w, b, dy2)                       # eager work between the replays
        xs.copy_(x2), dys.copy_(dy2)
        for gr, out in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_layer_norm_past_two_to_the_31_elements():
    rows, cols = (1 << 20) + 5, 2051
    assert rows * cols > 1 << 31
    g = torch.Generator(device=DEV).manual_seed(31)
    x, dy = (torch.randn(rows, cols, generator=g, device=DEV, dtype=F16) for _ in range(2))
    w, b = (torch.randn(cols, generator=g, device=DEV, dtype=F16) for _ in range(2))
    from gan_flow_amd.lib.layers import layer_norm
    x.requires_grad_()
    y = layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, dy)
    for part in (slice(0, 3), slice(rows // 2, rows // 2 + 40), slice(rows - 60, rows)):
        for name, got, (want, tol) in zip(("y", "dx"), (y.detach()[part], dx[part]), norm_reference(x.detach()[part], w, b, 1e-5, dy[part], F16, F16)):
            check(got, want, tol, "%s, rows %s" % (name, part))


# ---- Newton-Schulz orthogonalisation --------------------------------------------------------------------------------------

COEF = (3.4445, -4.7750, 2.0315)


def ns_reference(g, steps=5, coefficients=COEF, eps=1e-7):
    """(X, tolerance on |error|_F) of one matrix in 64 bits.  The tolerance is the deviation of a second 64-bit run in which
    every product P Q is disturbed by normal noise of 4 u |P||Q| and every operand by 2 u relative: what operands of 23 bits,
    the dropped low x low products (2^-22) and fp32 sums of errors of random sign leave, with a factor 2 on top."""
    gen = torch.Generator(device=g.device).manual_seed(1234)
    noise = lambda t: torch.randn(t.shape, generator=gen, device=t.device, dtype=torch.float64)  # noqa: E731
    tall = g.shape[0] > g.shape[1]
    x = (g.t() if tall else g).double().contiguous()
    x = x / (x.norm() + eps)
    z = x * (1 + 2 * U * noise(x))
    coefficients = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients

    def product(p, q):
        p, q = p * (1 + 2 * U * noise(p)), q * (1 + 2 * U * noise(q))
        r = p @ q
        return r + 4 * U * noise(r) * (p.abs() @ q.abs())

    for a, b, c in coefficients:
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
        s = product(z, z.t().contiguous())
        z = product(a * torch.eye(len(s), device=s.device, dtype=s.dtype) + b * s + c * product(s, s), z)
    tol = 2 * (z - x).norm() + 8 * U * x.norm()
    return (x.t() if tall else x), tol.item()


def check_ns(got, g, what="", **kw):
    want, tol = ns_reference(g, **kw)
    assert got.dtype == g.dtype and got.shape == g.shape
    err = (got.double() - want).norm().item()
    allowed = tol + rounded(want, g.dtype).norm().item()
    assert err <= allowed, "%s: |error|_F %g, %g allowed (|X|_F %g)" % (what, err, allowed, want.norm())


MATRICES = [(1, 1), (1, 5), (5, 1), (2, 64), (64, 2), (16, 16), (63, 65), (64, 64), (65, 64), (64, 66), (40, 300), (300, 40), (128, 128),
            (129, 70), (100, 256), (256, 256), (257, 255), (500, 130), (384, 640), (1000, 333)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: IDS[t])
@pytest.mark.parametrize("rows, cols", MATRICES)
def test_orthogonalize(rows, cols, dtype):
    from gan_flow_amd.lib.optim import orthogonalize
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows * 1000 + cols)).to(DEV, dtype)
    check_ns(orthogonalize(g), g)


@pytest.mark.parametrize("count, rows, cols", [(40, 130, 260), (9, 700, 500), (3, 1290, 520), (4, 1990, 2100), (1, 2900, 2950), (1, 300, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: IDS[t])
def test_orthogonalize_larger_launches(count, rows, cols, dtype):
    """Enough work for every tile the products are built for, at sizes that fill none of them."""
    from gan_flow_amd.lib.optim import orthogonalize
    g = torch.randn(count, rows, cols, generator=torch.Generator().manual_seed(count)).to(DEV, dtype)
    out = orthogonalize(g)
    for i in sorted({0, count // 2, count - 1}):
        check_ns(out[i], g[i], "matrix %d" % i)


@pytest.mark.parametrize("count, rows, cols", [(1, 50, 5000), (2, 5001, 64), (3, 64, 2100), (7, 1030, 3), (1, 33, 65536), (64, 20, 130)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: IDS[t])
def test_orthogonalize_of_short_sides(count, rows, cols, dtype):
    """One side of at most a tile, the other of many: several tiles a workgroup, workgroups without a full share."""
    from gan_flow_amd.lib.optim import orthogonalize
    wide = torch.randn(count, rows, cols + 3, generator=torch.Generator().manual_seed(count + rows)).to(DEV, dtype)
    for g in (wide[..., :cols].contiguous(), wide[..., 3:]):
        out = orthogonalize(g)
        for i in sorted({0, count // 2, count - 1}):
            check_ns(out[i], g[i], "matrix %d" % i)


@pytest.mark.parametrize("rows, cols", [(40, 900), (900, 40), (3, 300)])
@pytest.mark.parametrize("steps, coefficients", [(1, COEF), (2, COEF), (9, (2.0, -1.5, 0.5))])
def test_orthogonalize_of_short_sides_in_other_steps(rows, cols, steps, coefficients):
    from gan_flow_amd.lib.optim import orthogonalize
    gen = torch.Generator().manual_seed(rows)
    for scale in (1.0, 1e-12):                                # (the second far below eps)
        g = (torch.randn(2, rows, cols, generator=gen) * scale).to(DEV)
        out = orthogonalize(g, steps, coefficients)
        for i in range(2):
            check_ns(out[i], g[i], "matrix %d, scale %g" % (i, scale), steps=steps, coefficients=coefficients)


@pytest.mark.parametrize("rows, cols", [(200, 300), (300, 140), (64, 64), (40, 500)])
@pytest.mark.parametrize("dtype, scales", [(F16, (1.0, 1e-4, 6000.0)), (BF16, (1.0, 1e-9, 1e-30, 1e30))], ids=["fp16", "bf16"])
def test_orthogonalize_of_16_bit_matrices_of_any_scale(rows, cols, dtype, scales):
    from gan_flow_amd.lib.optim import orthogonalize
    gen = torch.Generator().manual_seed(rows)
    for scale in scales:
        g = (torch.randn(rows, cols, generator=gen) * scale).to(DEV, dtype)
        for steps in (1, 5):
            check_ns(orthogonalize(g, steps), g, "scale %g, %d steps" % (scale, steps), steps=steps)


@pytest.mark.parametrize("rows, cols", [(64, 64), (33, 50), (200, 90), (320, 320)])
def test_orthogonalize_batches_and_strides(rows, cols):
    from gan_flow_amd.lib.optim import orthogonalize
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 3, rows, cols + 7, generator=gen).to(DEV)
    for g in (wide[..., :cols], wide[..., 3:cols + 3], wide[0, :, :, :cols].transpose(1, 2), wide[:, 1, :, 1:cols + 1]):
        out = orthogonalize(g)
        flat, oflat = g.reshape((-1,) + g.shape[-2:]), out.reshape((-1,) + out.shape[-2:])
        assert out.shape == g.shape
        for i in range(len(flat)):
            check_ns(oflat[i], flat[i], "matrix %d" % i)


@pytest.mark.parametrize("rows, cols", [(64, 64), (150, 90)])
def test_orthogonalize_edges(rows, cols):
    from gan_flow_amd.lib.optim import orthogonalize
    gen = torch.Generator().manual_seed(4)
    g = torch.randn(6, rows, cols, generator=gen).to(DEV)
    g[1] = 0
    g[2] = g[2, :, :1] * g[2, :1, :]                        # rank one
    g[3] *= 1e30                                            # its squares overflow fp32
    g[4] *= 1e-30                                           # smaller than eps: X0 is nearly g / eps
    g[5, 0, 1:] = 0
    out = orthogonalize(g)
    assert out[1].eq(0).all()
    for i in (0, 2, 3, 4, 5):
        check_ns(out[i], g[i], "matrix %d" % i)
    for bad in (float("nan"), float("inf"), float("-inf")):
        g2 = g.clone()
        g2[2, 3, 4] = bad
        out2 = orthogonalize(g2)
        assert out2[2].isnan().all() and torch.equal(out2[[0, 1, 3, 4, 5]], out[[0, 1, 3, 4, 5]])
    assert orthogonalize(g[:0]).shape == (0, rows, cols) and orthogonalize(g[:, :0]).shape == (6, 0, cols)


@pytest.mark.parametrize("rows, cols", [(64, 64), (96, 200)])
def test_orthogonalize_other_polynomials(rows, cols):
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import orthogonalize
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(5)).to(DEV)
    for kw in (dict(steps=1), dict(steps=2), dict(steps=12, coefficients=(1.5, -0.5, 0.0)), dict(steps=3, eps=0.5),
               dict(steps=3, coefficients=[(4.0, -6.0, 2.5), (3.0, -3.5, 1.4), (1.5, -0.5, 0.0)])):
        check_ns(orthogonalize(g, **kw), g, str(kw), **kw)
    x = orthogonalize(g, steps=16, coefficients=(1.875, -1.25, 0.375)).double()   # converges: U V^T
    s = torch.linalg.svdvals(g.double() / g.double().norm())
    if s.min() > 2e-3:                                                            # (1.875^16 = 2.3e4 lifts that to 1)
        p = x @ x.t()
        assert (p - torch.eye(len(p), device=DEV)).norm() <= 1e-3
    with pytest.raises(CnfError, match="diverge"):
        orthogonalize(g, coefficients=(9.0, 0.0, 0.0))
    with pytest.raises(CnfError):
        orthogonalize(g[0])
    with pytest.raises(CnfError):
        orthogonalize(g.double())


def test_orthogonalize_many_matrices_in_place_and_deterministic():
    from gan_flow_amd import _native as nat
    from gan_flow_amd.lib.optim import orthogonalize
    g = torch.randn(150, 20, 24, generator=torch.Generator().manual_seed(6)).to(DEV)   # three calls of at most 64
    out = orthogonalize(g)
    for i in (0, 63, 64, 149):
        check_ns(out[i], g[i], "matrix %d" % i)
        assert torch.equal(orthogonalize(g[i]), out[i])
    assert torch.equal(orthogonalize(g), out)
    work = g[:5].clone()
    nat.orthogonalize(list(work), list(work), nat.newton_schulz())
    assert torch.equal(work, out[:5])


# ---- the Muon update ------------------------------------------------------------------------------------------------------

def muon_reference(w, g, m, lr, momentum, nesterov, wd, scale, dtype):
    w, g, m = w.double(), g.double(), m.double()
    m1 = momentum * m + g
    u = g + momentum * m1 if nesterov else m1
    x, tol = ns_reference(u)
    w1 = (1 - lr * wd) * w - lr * scale * x
    # the momentum and its factor are rounded, twice under Nesterov: the matrix that is iterated is off by about 4 u relative, which
    # the five steps lift at most 3.4445^5 = 485-fold: 2048 u |X| on top
    return w1, lr * scale * (tol + 2048 * U * x.norm().item()) + (3 * U * w.abs()).norm().item() + rounded(w1, dtype).norm().item(), m1


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: IDS[t])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("rows, cols", [(64, 64), (2, 64), (64, 2), (1, 9), (48, 31), (256, 256), (130, 400), (400, 130)])
def test_muon_step(rows, cols, nesterov, dtype):
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(rows + 31 * cols)
    kw = dict(lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.05, scale=0.7)
    w, g, m = (torch.randn(3, rows, cols, generator=gen).to(DEV) for _ in range(3))
    w, g = w.to(dtype), g.to(dtype)
    w0, g0, m0 = w.clone(), g.clone(), m.clone()
    muon_step(list(w), list(g), list(m), **kw)
    assert torch.equal(g, g0)
    for i in range(3):
        want, tol, m1 = muon_reference(w0[i], g0[i], m0[i], kw["lr"], kw["momentum"], nesterov, kw["weight_decay"], kw["scale"], dtype)
        check(m[i], m1, 3 * U * (m0[i].double().abs() + g0[i].double().abs()), "momentum")
        err = (w[i].double() - want).norm().item()
        assert err <= tol, "|error|_F %g, %g allowed" % (err, tol)


def test_muon_step_of_strided_blocks_leaves_the_rest():
    """Parameters that are blocks of wider matrices (padded hidden widths), of several shapes in one call."""
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(8)
    bufs = [torch.randn(3, 80, 96, generator=gen).to(DEV) for _ in range(3)]
    before = [b.clone() for b in bufs]
    block = lambda b: [b[0, :64, :64], b[1, 8:72, 16:80], b[2, :33, :90]]  # noqa: E731
    muon_step(*[block(b) for b in bufs], lr=0.1, scale=1.0)
    mask = torch.zeros_like(bufs[0], dtype=torch.bool)
    for t in block(mask):
        t.fill_(True)
    assert torch.equal(bufs[1], before[1])
    for i in (0, 2):
        assert torch.equal(bufs[i][~mask], before[i][~mask]) and not torch.equal(bufs[i][mask], before[i][mask])
    for w, w0, g0, m0 in zip(block(bufs[0]), block(before[0]), block(before[1]), block(before[2])):
        want, tol, _ = muon_reference(w0, g0, m0, 0.1, 0.95, True, 0.1, 1.0, F32)
        assert (w.double() - want).norm().item() <= tol


def test_muon_step_in_a_buffer_past_two_to_the_31_elements():
    from gan_flow_amd.lib.optim import muon_step
    rows, ld, cols = 33100, 65536, 48
    assert rows * ld > 1 << 31
    gen = torch.Generator(device=DEV).manual_seed(32)
    w, g, m = (torch.zeros(rows, ld, dtype=t, device=DEV)[:, 5:5 + cols] for t in (F16, F16, F32))
    for t in (w, g, m):
        t.copy_(torch.randn(rows, cols, generator=gen, device=DEV))
    w0, m0 = w.clone(), m.clone()
    muon_step([w], [g], [m], lr=0.1, weight_decay=0.05, scale=3.0)
    want, tol, m1 = muon_reference(w0, g, m0, 0.1, 0.95, True, 0.05, 3.0, F16)
    check(m, m1, 3 * U * (m0.double().abs() + g.double().abs()), "momentum")
    assert (w.double() - want).norm().item() <= tol


def test_muon_step_tells_autograd_and_refuses_a_momentum_as_gradient():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import muon_step
    w, m = torch.randn(70, 80, device=DEV), torch.zeros(70, 80, device=DEV)
    g = torch.randn(70, 80, device=DEV)
    before = w._version, m._version, g._version
    muon_step([w], [g], [m])
    assert w._version > before[0] and m._version > before[1] and g._version == before[2]
    with pytest.raises(CnfError, match="also a momentum"):
        muon_step([w], [m], [m])
    with pytest.raises(CnfError, match="given twice"):
        muon_step([w], [g], [w])
    with torch.inference_mode():
        muon_step([w.clone()], [g.clone()], [m.clone()])


def test_muon_step_guard_and_refusals():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(9)
    for shape in ((64, 64), (100, 70)):
        w, g, m = (torch.randn(*shape, generator=gen).to(DEV) for _ in range(3))
        w0, m0 = w.clone(), m.clone()
        words = torch.zeros(8, dtype=torch.int32, device=DEV)
        words[0] = 2
        muon_step([w], [g], [m], guard=words)
        assert torch.equal(w, w0) and torch.equal(m, m0)
        words.zero_()
        muon_step([w], [g], [m], guard=words)
        assert not torch.equal(w, w0) and not torch.equal(m, m0)
        muon_step([w[:0]], [g[:0]], [m[:0]])
        for bad in ((([w, w], [g, g], [m, m.clone()])), ([w, w.clone()], [g, g], [m, m]), ([w], [g.half()], [m]), ([w], [g], [m.half()]),
                    ([w], [g[:-1]], [m]), ([w.t().contiguous().t()], [g], [m]), ([w[0]], [g[0]], [m[0]]), ([w[:1].expand(4, shape[1])], [g[:4]], [m[:4]])):
            with pytest.raises(CnfError):
                muon_step(*bad)
        with pytest.raises(CnfError):
            muon_step([w], [g], [m], momentum=1.0)


def test_muon_optimizer_groups_state_and_resume():
    from gan_flow_amd.lib.optim import Muon, muon_step
    gen = torch.Generator().manual_seed(10)
    shapes = [(64, 64), (64, 64), (32, 64), (2, 64)]
    params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(DEV)) for s in shapes]
    ref = [p.detach().clone() for p in params]
    mom = [torch.zeros_like(r) for r in ref]
    opt = Muon(params, lr=0.02, adjust_lr="match_rms_adamw")
    for it in range(4):
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen).to(DEV)
        if it == 2:                                              # a resumed optimizer goes on where the first stopped
            state = opt.state_dict()
            opt = Muon(params, lr=0.5)
            opt.load_state_dict(state)
        for r, p, m in zip(ref, params, mom):
            muon_step([r], [p.grad], [m], lr=0.02, scale=0.2 * max(r.shape) ** 0.5)
        assert opt.step(lambda: it) == it
        assert all(torch.equal(r, p.detach()) for r, p in zip(ref, params))
    params[1].grad = None
    keep = params[1].detach().clone()
    opt.step()
    assert torch.equal(keep, params[1].detach())
    half = torch.nn.Parameter(torch.randn(16, 16, generator=gen).to(DEV, BF16))
    half.grad = torch.randn(16, 16, generator=gen).to(DEV, BF16)
    o = Muon([half])
    o.step()
    o.load_state_dict(o.state_dict())
    assert o.state[half]["momentum_buffer"].dtype == F32
    o.step()


def test_muon_captured_twice_and_replayed():
    """Two captured graphs of updates, replayed in turn with eager work between, against eager updates."""
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(11)
    for shape in ((64, 64), (200, 120)):
        w, g, m = (torch.randn(2, *shape, generator=gen).to(DEV) for _ in range(3))
        we, me = w.clone(), m.clone()
        muon_step(list(w), list(g), list(m)), muon_step(list(we), list(g), list(me))
        torch.cuda.synchronize()
        graphs = []
        for i in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                muon_step([w[i]], [g[i]], [m[i]])
            graphs.append(gr)
        for _ in range(3):
            for gr in graphs:
                gr.replay()
            g2 = torch.randn(2, *shape, generator=gen).to(DEV)
            muon_step(list(we), list(g), list(me))
            torch.cuda.synchronize()
            assert torch.equal(w, we) and torch.equal(m, me)
            g.copy_(g2)


def test_normalised_network_trained_with_muon():
    """The operators together, as a training step uses them: a conditioner of two hidden matrices with a layer norm between,
    its matrices stepped by Muon and its vectors by Adam; the first step against 64 bits, and the loss's gradients with it."""
    from gan_flow_amd.lib.layers import LayerNorm
    from gan_flow_amd.lib.optim import Muon
    gen = torch.Generator().manual_seed(12)
    rows, d, h = 256, 64, 96
    x, t = (torch.randn(rows, d, generator=gen).to(DEV) for _ in range(2))
    w1, w2 = (torch.nn.Parameter((torch.randn(s, generator=gen) / s[1] ** 0.5).to(DEV)) for s in ((h, d), (d, h)))
    norm = LayerNorm(h).to(DEV)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.2 * torch.randn(h, generator=gen)), norm.bias.copy_(0.2 * torch.randn(h, generator=gen))

    def forward(a, b, g, s, f, dt):
        return ((torch.tanh(f((x.to(dt) @ a.t()), g, s)) @ b.t() - t.to(dt)).square().mean())

    def plain(v, g, s):
        mean = v.mean(1, keepdim=True)
        return (v - mean) / ((v - mean).square().mean(1, keepdim=True) + norm.eps).sqrt() * g + s

    leaves = [w1, w2, norm.weight, norm.bias]
    exact = [p.detach().double().requires_grad_() for p in leaves]
    want = torch.autograd.grad(forward(*exact, plain, torch.float64), exact)
    muon, adam = Muon([w1, w2], lr=0.02), torch.optim.Adam([norm.weight, norm.bias], lr=1e-3)
    forward(*leaves, lambda v, g, s: norm(v), F32).backward()
    for p, g64 in zip(leaves, want):
        # four layers of fp32 sums of at most 256 terms, forward and backward: 2 * 4 * 256 u, twice for the functions between
        assert (p.grad.double() - g64).norm() <= 4096 * U * g64.norm()
    before = [p.detach().clone() for p in (w1, w2)]
    muon.step(), adam.step()
    for p, b, name in zip((w1, w2), before, "12"):
        w, tol, _ = muon_reference(b, p.grad, torch.zeros_like(b), 0.02, 0.95, True, 0.1, max(1.0, b.shape[0] / b.shape[1]) ** 0.5, F32)
        assert (p.detach().double() - w).norm().item() <= tol, name
    for _ in range(3):
        muon.zero_grad(), adam.zero_grad()
        loss = forward(*leaves, lambda v, g, s: norm(v), F32)
        loss.backward()
        muon.step(), adam.step()
    assert torch.isfinite(loss)


def test_calls_on_two_streams_at_once():
    """Two streams busy with calls of their own, each result the bits of the same call alone."""
    from gan_flow_amd.lib.layers import layer_norm
    from gan_flow_amd.lib.optim import muon_step, orthogonalize
    gen = torch.Generator().manual_seed(77)
    gs = [torch.randn(c, r, n, generator=gen).to(DEV) for c, r, n in ((3, 300, 200), (2, 64, 40), (1, 700, 900))]
    x = torch.randn(500, 900, generator=gen).to(DEV)
    w, m = torch.randn(300, 200, generator=gen).to(DEV), torch.randn(300, 200, generator=gen).to(DEV)

    def work():
        w1, m1 = w.clone(), m.clone()
        muon_step([w1], [gs[0][0]], [m1])
        return [orthogonalize(g) for g in gs] + [layer_norm(x), w1, m1]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_training_step_of_a_normalised_layer_captured_and_replayed():
    """Forward, backward through autograd and the Muon update of one layer in one captured graph, against the eager steps."""
    from gan_flow_amd.lib.layers import layer_norm
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(78)
    w0, s0, b0 = torch.randn(96, 130, generator=gen).to(DEV) / 10, torch.ones(96, device=DEV), torch.zeros(96, device=DEV)
    xs = [torch.randn(200, 130, generator=gen).to(DEV) for _ in range(4)]
    dy = torch.randn(200, 96, generator=gen).to(DEV)

    def step(x, w, s, b, m):
        y = layer_norm(x @ w.t(), s, b)
        gw, gs, gb = torch.autograd.grad(y, (w, s, b), dy)
        with torch.no_grad():
            muon_step([w], [gw], [m], lr=0.02)
            s.sub_(gs, alpha=0.01), b.sub_(gb, alpha=0.01)
        return y.detach()

    def leaves():
        return [t.clone().requires_grad_() for t in (w0, s0, b0)] + [torch.zeros_like(w0)]

    eager = leaves()
    want = [(step(x, *eager), [t.detach().clone() for t in eager]) for x in xs]
    mine, x = leaves(), torch.empty_like(xs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs[0], *mine)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, *mine)
    with torch.no_grad():
        for t, v in zip(mine, (w0, s0, b0, torch.zeros_like(w0))):
            t.copy_(v)
    for k, xk in enumerate(xs):
        x.copy_(xk)
        graph.replay()
        torch.cuda.synchronize()
        layer_norm(xk)                                        # eager work between the replays
        assert torch.equal(out, want[k][0])
        assert all(torch.equal(t.detach(), v) for t, v in zip(mine, want[k][1]))


# ---- no less exact than plain fp32 ----------------------------------------------------------------------------------------

def _spectrum(kind, count, rows, cols):
    """Normal matrices, gradients (a decaying spectrum over noise), or singular values over `kind` decades; 64 bits."""
    gen = torch.Generator(device=DEV).manual_seed(rows + cols)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV, dtype=torch.float64)  # noqa: E731
    m = min(rows, cols)
    if kind == "normal":
        g = randn(count, m, max(rows, cols))
    elif kind == "gradient":
        g = (randn(count, m, m) * torch.logspace(0, -3, m, device=DEV)) @ randn(count, m, max(rows, cols)) / m ** 0.5 + 0.1 * randn(count, m, max(rows, cols))
    else:
        u, v = torch.linalg.qr(randn(count, m, m))[0], torch.linalg.qr(randn(count, max(rows, cols), m))[0]
        g = (u * torch.logspace(0, -kind, m, device=DEV)) @ v.transpose(1, 2).contiguous()
    return (g if rows <= cols else g.transpose(1, 2)).contiguous()


def _plain(g, steps=5):
    x = g.transpose(1, 2).contiguous() if g.shape[1] > g.shape[2] else g
    x = x / (x.double().square().sum((1, 2), keepdim=True).sqrt() + 1e-7).to(x.dtype)
    a, b, c = COEF
    for _ in range(steps):
        s = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(1, 2) if g.shape[1] > g.shape[2] else x


@pytest.mark.parametrize("kind", ["normal", "gradient", 2, 3])
@pytest.mark.parametrize("count, rows, cols", [(4, 80, 5000), (4, 4000, 100), (40, 130, 260), (2, 300, 9000), (8, 200, 800), (2, 512, 1100), (2, 900, 260)])
def test_orthogonalize_is_as_exact_as_plain_fp32(count, rows, cols, kind):
    """Operands of 23 bits round at most twice what those of 24 do, and everything else is fp32 in both: twice the error of the same
    iteration in fp32 tensor operations is allowed."""
    from gan_flow_amd.lib.optim import orthogonalize
    g = _spectrum(kind, count, rows, cols).float()
    want = _plain(g.double())
    err = lambda x: ((x.double() - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))).mean().item()  # noqa: E731
    mine, plain = err(orthogonalize(g)), err(_plain(g))
    assert mine <= 2 * plain, "%g, and %g of the plain form" % (mine, plain)


def test_operators_refuse_forward_mode():
    from torch.autograd import forward_ad
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.layers import layer_norm
    from gan_flow_amd.lib.optim import orthogonalize
    x = torch.randn(70, 80, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = layer_norm(x), orthogonalize(x)
    with forward_ad.dual_level():
        assert torch.equal(layer_norm(x), want[0]) and torch.equal(orthogonalize(x), want[1])
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            layer_norm(dual)
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            layer_norm(x, dual[0])
        with pytest.raises(CnfError, match="tangent"):
            orthogonalize(dual)


def test_layer_norm_of_an_empty_batch_without_weight_gradients():
    from gan_flow_amd.lib.layers import layer_norm
    w, b = torch.ones(12, device=DEV), torch.zeros(12, device=DEV)
    for shape in ((0, 12), (2, 0, 12)):
        for args in ((None, None), (w, b)):
            x = torch.empty(shape, device=DEV, requires_grad=True)
            y = layer_norm(x, *args)
            y.sum().backward()
            assert y.shape == shape and x.grad.shape == shape
    x = torch.empty(0, 12, device=DEV)
    for lw, lb in ((w.clone().requires_grad_(), b), (w, b.clone().requires_grad_())):
        layer_norm(x, lw, lb).sum().backward()
        assert all(t.grad.eq(0).all() for t in (lw, lb) if t.requires_grad)


def test_a_refused_muon_update_changes_nothing():
    """One matrix among several that cannot be updated, whatever its place: the others are left as they were."""
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import Muon, muon_step
    gen = torch.Generator().manual_seed(41)
    make = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    good = [(make(64, 64), make(64, 64), make(64, 64)), (make(70, 90), make(70, 90), make(70, 90))]
    before = [[t.clone() for t in three] for three in good]
    w, g, m = make(48, 32), make(48, 32), make(48, 32)
    turned = lambda t: t.t().contiguous().t()  # noqa: E731
    for bad in ((turned(w), g, m), (w, g, turned(m)), (w, g.half(), m), (w, g, m.half()), (w.double(), g.double(), m), (w, g[:-1], m), (w, g, m[:-1]),
                (w, g, good[0][2]), (w, m, m), (torch.zeros(1, 65537, device=DEV),) * 3):
        for at in range(3):
            lists = [list(t) for t in zip(*(good[:at] + [bad] + good[at:]))]
            with pytest.raises(CnfError):
                muon_step(*lists)
    assert all(torch.equal(t, s) for three, saved in zip(good, before) for t, s in zip(three, saved))
    params = [torch.nn.Parameter(t) for t in (make(64, 64), turned(make(48, 32)), make(70, 90))]
    opt = Muon(params[:1])
    opt.add_param_group(dict(params=params[1:]))
    for p in params:
        p.grad = make(*p.shape)
    saved = [p.detach().clone() for p in params]
    with pytest.raises(CnfError, match="contiguous"):
        opt.step()
    assert all(torch.equal(p, s) for p, s in zip(params, saved))
    assert all(opt.state[p]["momentum_buffer"].eq(0).all() for p in params)
    params[1].grad = None
    opt.step()
    assert [torch.equal(p, s) for p, s in zip(params, saved)] == [False, True, False]


def test_the_binding_and_the_optimizer_take_the_same_step():
    from gan_flow_amd import _native as nat
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(42)
    for shape in ((3, 64, 64), (2, 1, 9), (2, 100, 300)):
        w, g, m = (torch.randn(shape, generator=gen).to(DEV) for _ in range(3))
        w2, m2 = w.clone(), m.clone()
        muon_step(list(w), list(g), list(m), lr=0.1, scale=0.5)
        nat.muon_step(w2, g, m2, nat.newton_schulz(), lr=0.1, scale=0.5)
        assert torch.equal(w, w2) and torch.equal(m, m2)


def test_muon_step_refuses_another_matrixs_parameter_as_gradient():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(43)
    for a, b in (((64, 64), (64, 64)), ((100, 80), (100, 80))):
        w, v = (torch.randn(s, generator=gen).to(DEV) for s in (a, b))
        m = [torch.zeros_like(w), torch.zeros_like(v)]
        for g in ([v, v.clone()], [w.clone(), w], [v, w]):
            with pytest.raises(CnfError, match="another matrix's parameter"):
                muon_step([w, v], g, m)
        w0, v0 = w.clone(), v.clone()
        muon_step([w, v], [w, v], m)                           # its own: decay along the parameter itself
        want = [t.clone() for t in (w0, v0)]
        muon_step(want, [w0, v0], [torch.zeros_like(w), torch.zeros_like(v)])
        assert torch.equal(w, want[0]) and torch.equal(v, want[1])


def test_layer_norm_refuses_what_has_no_features_or_no_tensors():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.layers import layer_norm
    for x in (torch.empty(2, 3, 0), torch.empty(0), torch.empty(0, 0)):
        with pytest.raises(CnfError, match="cols > 0"):
            layer_norm(x.to(DEV))
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    for args in (([1.0] * 8, None), (None, 1.0), (2.0, None)):
        with pytest.raises(CnfError, match="HIP device"):
            layer_norm(x, *args)
    for shape in ((3, 0, 8), (0, 3, 8), (0, 8), (2, 0, 0, 8)):
        assert layer_norm(torch.empty(shape, device=DEV)).shape == shape


# ---- every kernel of the larger products ----------------------------------------------------------------------------------

# (count, rows, cols): (steps together, tiles of X X^T, of the other symmetric products, of the products with X)
PLANS = {(12, 768, 768): (0, 128, 128, 128), (40, 515, 523): (0, 192, 192, 128), (16, 1000, 1000): (0, 256, 256, 256), (40, 370, 555): (0, 128, 128, 192),
         (8, 1010, 500): (0, 64, 64, 128), (6, 460, 2760): (1, 64, 64, 256), (40, 1120, 280): (1, 64, 128, 128), (1, 4000, 4030): (0, 192, 192, 256),
         (12, 310, 1860): (1, 64, 64, 192)}


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: IDS[t])
@pytest.mark.parametrize("shape", PLANS)
def test_orthogonalize_through_every_tile(shape, dtype):
    """16-bit matrices take the kernels of one and two products of pieces in their first step."""
    from gan_flow_amd import _native as nat
    from gan_flow_amd.lib.optim import orthogonalize
    count, rows, cols = shape
    assert nat.matrix_plan(*shape) == (2,) + PLANS[shape]
    gen = torch.Generator(device=DEV).manual_seed(rows)
    wide = torch.randn(count, rows, cols + 2, generator=gen, device=DEV)
    wide[..., 0] *= 30.0                                       # one direction far above the others
    wide = wide.to(dtype)
    for g in (wide[..., :cols].contiguous(), wide[..., 1:cols + 1]) if count * rows * cols < 1 << 23 else (wide[..., :cols].contiguous(),):
        out = orthogonalize(g)
        for i in sorted({0, count - 1}):
            check_ns(out[i], g[i], "matrix %d" % i)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: IDS[t])
@pytest.mark.parametrize("shape", [s for s in PLANS if s[0] > 1])
def test_muon_step_through_every_tile(shape, dtype):
    """Parameters in rows of wider buffers, under a guard: a failed solve changes nothing, the next one everything it should."""
    from gan_flow_amd import _native as nat
    from gan_flow_amd.lib.optim import muon_step
    count, rows, cols = shape
    assert nat.matrix_plan(*shape) == (2,) + PLANS[shape]
    gen = torch.Generator(device=DEV).manual_seed(cols)
    wide = torch.randn(count, rows, cols + 5, generator=gen, device=DEV).to(dtype)
    g, m = torch.randn(count, rows, cols, generator=gen, device=DEV).to(dtype), torch.randn(count, rows, cols, generator=gen, device=DEV)
    w = wide[..., 2:cols + 2]
    wide0, m0 = wide.clone(), m.clone()
    w0 = wide0[..., 2:cols + 2]
    words = torch.zeros(8, dtype=torch.int32, device=DEV)
    words[0] = 2
    kw = dict(lr=0.02, momentum=0.9, weight_decay=0.05, scale=0.7, guard=words)
    muon_step(list(w), list(g), list(m), **kw)
    assert torch.equal(wide, wide0) and torch.equal(m, m0)
    words.zero_()
    muon_step(list(w), list(g), list(m), **kw)
    assert torch.equal(wide[..., :2], wide0[..., :2]) and torch.equal(wide[..., cols + 2:], wide0[..., cols + 2:])
    for i in (0, count - 1):
        want, tol, m1 = muon_reference(w0[i], g[i], m0[i], 0.02, 0.9, True, 0.05, 0.7, dtype)
        check(m[i], m1, 3 * U * (m0[i].double().abs() + g[i].double().abs()), "momentum")
        err = (w[i].double() - want).norm().item()
        assert err <= tol, "matrix %d: |error|_F %g, %g allowed" % (i, err, tol)


@pytest.mark.parametrize("shape", [(3, 40, 900), (2, 900, 40), (2, 7, 65)])
def test_muon_step_of_short_sides_under_a_guard(shape):
    from gan_flow_amd.lib.optim import muon_step
    gen = torch.Generator().manual_seed(44)
    for dtype in (F32, F16, BF16):
        w, g, m = (torch.randn(shape, generator=gen).to(DEV) for _ in range(3))
        w, g = w.to(dtype), g.to(dtype)
        w0, m0 = w.clone(), m.clone()
        words = torch.ones(8, dtype=torch.int32, device=DEV)
        muon_step(list(w), list(g), list(m), lr=0.1, guard=words)
        assert torch.equal(w, w0) and torch.equal(m, m0)
        words.zero_()
        muon_step(list(w), list(g), list(m), lr=0.1, guard=words)
        for i in range(shape[0]):
            want, tol, m1 = muon_reference(w0[i], g[i], m0[i], 0.1, 0.95, True, 0.1, 1.0, dtype)
            check(m[i], m1, 3 * U * (m0[i].double().abs() + g[i].double().abs()), "momentum")
            assert (w[i].double() - want).norm().item() <= tol


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: IDS[t])
@pytest.mark.parametrize("rows, cols", [(64, 64), (40, 500), (500, 40), (150, 90), (1, 300), (220, 900)])
def test_orthogonalize_keeps_matrices_apart(rows, cols, dtype):
    """A NaN or an infinity makes its matrix NaN throughout and leaves the others in the call their bits."""
    from gan_flow_amd.lib.optim import muon_step, orthogonalize
    gen = torch.Generator().manual_seed(45)
    g = torch.randn(4, rows, cols, generator=gen).to(DEV, dtype)
    clean = orthogonalize(g)
    for bad in (float("nan"), float("inf"), float("-inf")):
        g2 = g.clone()
        g2[1, rows - 1, cols - 1] = bad
        g2[2, 0, cols // 2] = bad
        out = orthogonalize(g2)
        assert out[1:3].isnan().all() and torch.equal(out[[0, 3]], clean[[0, 3]])
        w, m = torch.zeros_like(g2), torch.zeros(g2.shape, device=DEV)
        muon_step(list(w), list(g2), list(m))
        assert w[1:3].isnan().all() and torch.isfinite(w[[0, 3]]).all() and torch.isfinite(m).sum() == m.numel() - 2


# ---- weight gradients over many rows --------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows, cols, dtype, wdtype", [
    (4099, 1001, F16, F32), (4097, 320, BF16, F32), (70001, 16, F32, F32), (20011, 64, BF16, BF16),   # a wave's lanes a row, more row groups than workgroups
    (1500, 2048, F32, F32), (1500, 2048, BF16, BF16), (2100, 1999, BF16, F32), (1300, 3001, F16, F16),
    (700, 8192, F32, F32), (700, 8192, F16, F16), (1100, 4100, F32, F32),                              # a workgroup a row, more rows than workgroups
    (300, 9000, F32, F32), (300, 9000, BF16, BF16), (20000, 8200, F16, F32)], ids=str)                 # long rows: several parts, the most parts
def test_layer_norm_weight_gradients_over_many_rows(rows, cols, dtype, wdtype):
    x, w, b, dy = norm_inputs(rows, cols, dtype, wdtype, 12)
    first = norm_both(x, w, b, dy)
    for name, got, (want, tol) in zip(("y", "dx", "dw", "db"), first, norm_reference(x, w, b, 1e-5, dy, dtype, wdtype)):
        check(got, want, tol, name)
    assert all(torch.equal(p, q) for p, q in zip(first, norm_both(x, w, b, dy)))


@pytest.mark.parametrize("shape", [(2, 40, 900), (2, 900, 230), (12, 700, 760)])
def test_matrix_products_captured_and_replayed(shape):
    """Orthogonalisation and update of every path in one captured graph, replayed with eager work between."""
    from gan_flow_amd.lib.optim import muon_step, orthogonalize
    gen = torch.Generator(device=DEV).manual_seed(46)
    new = lambda: torch.randn(shape, generator=gen, device=DEV)  # noqa: E731
    w, g, m = new(), new(), new()
    we, me = w.clone(), m.clone()
    muon_step(list(we), list(g), list(me)), orthogonalize(g)   # (before the capture, on copies that are put back)
    we.copy_(w), me.copy_(m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(list(w), list(g), list(m))
        out = orthogonalize(g)
    for _ in range(3):
        g.copy_(new())
        graph.replay()
        muon_step(list(we), list(g), list(me))
        want = orthogonalize(g)
        torch.cuda.synchronize()
        assert torch.equal(w, we) and torch.equal(m, me) and torch.equal(out, want)


def test_a_later_group_of_muon_that_would_diverge_leaves_the_first_alone():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import Muon
    gen = torch.Generator().manual_seed(47)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(DEV)) for s in ((64, 64), (70, 90))]
    opt = Muon(params[:1])
    opt.add_param_group(dict(params=params[1:]))
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(DEV)
    saved = [p.detach().clone() for p in params]
    for bad, error in ((dict(ns_coefficients=(9.0, 0.0, 0.0)), CnfError), (dict(lr=1e300, adjust_lr=1e300), ValueError), (dict(momentum=1.0), ValueError)):
        keep = dict(opt.param_groups[1])
        opt.param_groups[1].update(bad)
        with pytest.raises(error):
            opt.step()
        opt.param_groups[1].update(keep)
        assert all(torch.equal(p, s) for p, s in zip(params, saved))
    opt.step()
    assert not any(torch.equal(p, s) for p, s in zip(params, saved))
