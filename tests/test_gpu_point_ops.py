"""Rotary positions and the cross entropy of a linear head against their definitions in 64 bits, with bounds that follow from
the types: a rounding to a type with step eps is off by eps / 2 of the value at most."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24      # half a step of float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- rotary positions ----------------------------------------------------------------------------------------------------
def rotate64(x, pos, sections, base, style, sign=1.0):
    """(value, bound): the rotation in 64 bits, and how far a kernel may be off that holds the angle's fraction of a turn in 32
    bits (pi E of angle), takes sine and cosine within two steps (4 E), multiplies and adds in 32 bits (2 E) and rounds once."""
    x64 = x.detach().double().cpu()
    freq = torch.cat([base ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections if s]) if sum(sections) else torch.zeros(0, dtype=torch.float64)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    angle = (pos.double().cpu()[:, axis] * freq)[:, None, :]
    c, s = torch.cos(angle), torch.sin(angle) * sign
    r = len(axis)
    i1, i2 = (slice(0, r), slice(r, 2 * r)) if style == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    y, size = x64.clone(), torch.zeros_like(x64)
    y[..., i1], y[..., i2] = x64[..., i1] * c - x64[..., i2] * s, x64[..., i2] * c + x64[..., i1] * s
    size[..., i1] = size[..., i2] = x64[..., i1].abs() + x64[..., i2].abs()
    # the position times turns per unit: 2^-52 of the angle, and what the whole turns take of it
    lost = torch.zeros_like(x64)
    lost[..., i1] = lost[..., i2] = (angle.abs() * 2.0 ** -51).expand(-1, x64.shape[1], -1)
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    return y, size * (10 * E + lost) + torch.finfo(x.dtype).eps / 2 * y.abs() + tiny


def near(got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs() - bound
    assert not torch.isnan(off).any() and off.max().item() <= 0, (off.max().item(), (got - want).abs().max().item())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,kv,dim,sections,pos", [
    (1, 1, 0, 2, (1,), "i32"), (7, 3, 1, 10, (2, 3), "f32"), (65, 4, 4, 48, (8, 8, 8), "f32"), (300, 8, 2, 64, (10, 10, 10), "i64"),
    (33, 1, 1, 130, (5, 0, 7, 9), "f64"), (1030, 2, 1, 96, (48,), "i32"), (5, 40, 8, 256, (32, 32, 64), "i32"), (3, 2, 0, 8, (0,), "f32"),
    (2, 70, 70, 512, (256,), "f32")])
def test_rotary(pkg, dtype, style, tokens, heads, kv, dim, sections, pos):
    g = gen(tokens * 31 + dim)
    q = torch.randn((tokens, heads, dim), generator=g).to(dtype).cuda().requires_grad_()
    k = torch.randn((tokens, kv, dim), generator=g).to(dtype).cuda().requires_grad_() if kv else None
    kind = {"i32": torch.int32, "i64": torch.int64, "f32": torch.float32, "f64": torch.float64}[pos]
    p = (torch.randn((tokens, len(sections)), generator=g) * 50).to(kind).cuda()
    a, b = pkg.rotary_positions(q, p, sections, key=k, base=500.0, style=style)
    assert a.dtype == dtype and (b is None) == (k is None)
    for x, y in ((q, a), (k, b)):
        if x is None:
            continue
        near(y, *rotate64(x, p, sections, 500.0, style))
        up = torch.randn(y.shape, generator=g).to(dtype).cuda()
        back, = torch.autograd.grad(y, x, up, retain_graph=True)
        near(back, *rotate64(up, p, sections, 500.0, style, -1.0))


def test_rotary_gradient_against_differences(pkg):
    g = gen(5)
    x = torch.randn((9, 2, 12), generator=g).cuda().requires_grad_()
    p, up = torch.randn((9, 2), generator=g).cuda() * 7, torch.randn((9, 2, 12), generator=g).cuda()
    f = lambda v: (pkg.rotary_positions(v, p, (3, 2))[0].double() * up.double()).sum()  # noqa: E731
    got, = torch.autograd.grad(f(x), x)
    for t, h, e in ((0, 0, 0), (3, 1, 4), (8, 0, 11), (5, 1, 9)):
        step = torch.zeros_like(x)
        step[t, h, e] = 0.5
        # the map is linear: a difference of any length is exact but for 32-bit rounding of both sides, over a step of 1
        want = (f((x + step).detach()) - f((x - step).detach())).item()
        assert abs(got[t, h, e].item() - want) <= 64 * E * (up[t, h].abs().sum().item() * (x[t, h].abs().max().item() + 1))


def test_rotary_far_positions(pkg):
    p = torch.tensor([[0], [1], [161279], [2 ** 31 - 1], [-2 ** 31]], dtype=torch.int32)
    x = torch.randn((5, 1, 64), generator=gen(1))
    y, _ = pkg.rotary_positions(x.cuda(), p.cuda(), (32,))
    near(y, *rotate64(x, p, (32,), 10000.0, "half"))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotary_takes_strides(pkg, dtype):
    g = gen(3)
    fused = torch.randn((50, 6, 24), generator=g).to(dtype).cuda()
    rows = torch.randn((50, 4), generator=g).cuda() * 20      # points: x y z are a slice
    q, k = fused[:, :4], fused[:, 4:5]
    a, b = pkg.rotary_positions(q, rows[:, :3], (4, 4, 3), key=k)
    near(a, *rotate64(q, rows[:, :3], (4, 4, 3), 10000.0, "half"))
    near(b, *rotate64(k, rows[:, :3], (4, 4, 3), 10000.0, "half"))
    turned = fused[:, :4].transpose(1, 2).contiguous().transpose(1, 2)      # the last axis is not dense
    near(pkg.rotary_positions(turned, rows[:, :3], (4, 4, 3))[0], *rotate64(q, rows[:, :3], (4, 4, 3), 10000.0, "half"))
    by_head = fused[:, :4].transpose(0, 1).contiguous().transpose(0, 1)      # heads outside
    near(pkg.rotary_positions(by_head, rows[:, :3], (4, 4, 3), style="interleaved")[0], *rotate64(q, rows[:, :3], (4, 4, 3), 10000.0, "interleaved"))
    odd = fused.reshape(-1)[2:2 + 49 * 144].reshape(49, 6, 24)      # 4 (or 8) byte alignment
    near(pkg.rotary_positions(odd, rows[1:, 1:3], (4, 4))[0], *rotate64(odd, rows[1:, 1:3], (4, 4), 10000.0, "half"))
    wide = fused[:1].expand(50, 6, 24)      # one row for all tokens
    near(pkg.rotary_positions(wide, rows[:, :1], (12,))[0], *rotate64(wide, rows[:, :1], (12,), 10000.0, "half"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv,dim,sections", [(4, 2, 48, (8, 8, 8)), (3, 3, 34, (5, 5, 7)), (1, 0, 6, (3,)), (50, 7, 512, (100, 100, 56)), (5, 1, 2, (1,))])
def test_rotary_layouts_give_the_dense_result(pkg, dtype, heads, kv, dim, sections):
    """Slices of one projection, heads in front of tokens, one token for all, one head for all, rows that begin anywhere."""
    g = gen(heads * dim)
    tokens = 37
    pos = torch.randn((tokens, len(sections)), generator=g).cuda() * 50
    both = torch.randn((tokens, heads + 2 * kv + 1, dim + 2), generator=g).to(dtype).cuda()
    front = torch.randn((heads + kv, tokens, dim), generator=g).to(dtype).cuda().transpose(0, 1)
    whole = torch.randn((tokens, (heads + 2 * kv) * dim + 1), generator=g).to(dtype).cuda()[:, 1:].view(tokens, -1, dim) if dim > 2 else front
    for x in (both[:, 1:, :dim], both[:, 1:, 2:], both[:, :, 1:dim + 1], front, whole, both[:1, 1:, :dim].expand(tokens, -1, -1),
              both[:, :1, :dim].expand(-1, heads + kv, -1)):
        q, k = x[:, :heads], x[:, heads:heads + kv] if kv else None
        got = pkg.rotary_positions(q, pos, sections, key=k)
        want = pkg.rotary_positions(q.contiguous(), pos, sections, key=None if k is None else k.contiguous())
        assert torch.equal(got[0], want[0]) and (k is None or torch.equal(got[1], want[1]))
    if kv:      # the gradient of a view goes where the view's elements are
        x = both[:, 1:, :dim].detach().clone().requires_grad_()
        y, z = pkg.rotary_positions(x[:, :heads], pos, sections, key=x[:, heads:heads + kv])
        gy, gz = (torch.randn(t.shape, generator=g).to(dtype).cuda().transpose(0, 1).contiguous().transpose(0, 1) for t in (y, z))
        dx, = torch.autograd.grad((y, z), x, (gy, gz))
        turned = pkg.rotary_positions(torch.cat([gy, gz], 1).contiguous(), -pos, sections)[0]
        assert (dx[:, :heads + kv].float() - turned.float()).abs().max() <= 1e-6 and not dx[:, heads + kv:].any()


def test_rotary_of_nothing_and_not_a_number(pkg):
    q = torch.zeros((0, 2, 8), device="cuda", requires_grad=True)
    y, k = pkg.rotary_positions(q, torch.zeros((0, 1), device="cuda"), (4,))
    assert y.shape == (0, 2, 8) and k is None
    assert torch.autograd.grad(y.sum(), q)[0].shape == (0, 2, 8)
    x = torch.ones((2, 1, 8), device="cuda")
    x[0, 0, 7] = float("inf")      # behind the pairs: copied, touches nothing
    y, _ = pkg.rotary_positions(x, torch.tensor([[0.5], [float("nan")]], device="cuda"), (3,))
    assert torch.isfinite(y[0, 0, :7]).all() and y[0, 0, 7] == float("inf")
    assert torch.isnan(y[1, 0, :6]).all() and (y[1, 0, 6:] == 1).all()


# ---- cross entropy -------------------------------------------------------------------------------------------------------
def check_loss(pkg, n, v, d, dtype, bias=True, ignore=-100, reduction="mean", piece=0, target_type=torch.int64, share=0.2, spread=1.0, x=None, w=None,
               b="make", target=None, up=None, seed=0):
    """Loss and gradients against the definition in 64 bits, within the bounds of a kernel that sums in 32 bits and rounds dl to the
    inputs' type: a logit is off by e_l = (features + 16) E of the sum of its absolute products, a probability by twice that
    and 2^-20 (the exponent's base-2 argument, of at most 16 here, rounded to 32 bits), relative to itself."""
    g = gen(seed + n * 7 + v * 3 + d)
    if x is None:
        x = torch.randn((n, d), generator=g).to(dtype)
    if w is None:
        w = (torch.randn((v, d), generator=g) * spread * 2 / math.sqrt(d)).to(dtype)
    if isinstance(b, str):
        b = torch.randn((v,), generator=g).to(dtype) if bias else None
    if target is None:
        target = torch.randint(0, v, (n,), generator=g)
        target[torch.rand((n,), generator=g) < share] = ignore
    target = target.to(target_type)
    if up is None:
        up = torch.rand((n,), generator=g) * 3 - 1 if reduction == "none" else torch.tensor(2.5)
    ins = [None if t is None else t.cuda().requires_grad_() for t in (x, w, b)]
    loss = pkg.linear_cross_entropy(ins[0], ins[1], target.cuda(), bias=ins[2], ignore_index=ignore, reduction=reduction, piece=piece)
    assert loss.dtype == F32
    leaves = [t for t in ins if t is not None]
    got = torch.autograd.grad(loss, leaves, up.cuda())
    # ---- the definition, over the points that count
    x64, w64 = x.double(), w.double()
    b64 = torch.zeros(v, dtype=torch.float64) if b is None else b.double()
    keep = torch.nonzero(target.long() != ignore)[:, 0]
    xs, ts = x64[keep], target.long()[keep]
    logits = xs @ w64.t() + b64
    finite_b = torch.where(b64.abs() < 1e4, b64, 0)      # (masked classes take part in nothing)
    e_l = ((d + 16) * E * (xs.abs() @ w64.abs().t() + finite_b.abs() + 1)).amax(1, keepdim=True) if len(keep) else torch.zeros((0, 1), dtype=torch.float64)
    lse = torch.logsumexp(logits, 1, keepdim=True)
    each = lse[:, 0] - logits[torch.arange(len(keep)), ts]
    each_tol = 2 * e_l[:, 0] + 8 * E * (lse[:, 0].abs() + each.abs()) + 1e-30
    full, full_tol = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    full[keep], full_tol[keep] = each, each_tol
    count = max(1, len(keep)) if reduction == "mean" else 1
    if reduction == "none":
        near(loss, full, full_tol)
        weight = up.double()[keep][:, None]
    else:
        near(loss, full.sum() / count, full_tol.sum() / count + 2 * E * (full.abs().sum() / count))
        weight = up.double() / count * torch.ones((len(keep), 1), dtype=torch.float64)
    p = torch.exp(logits - lse)
    dl = p.clone()
    dl[torch.arange(len(keep)), ts] -= 1
    u = torch.finfo(dtype).eps / 2
    # float32 is held in planes (2^-25) and multiplied without the products below 2^-24 (three of them)
    u_dl = 2.0 ** -22 if dtype == F32 else u
    dl_tol = weight.abs() * (p * (2 * e_l + 2.0 ** -20) + u_dl * dl.abs())
    if dtype == F16:      # steps below the smallest normal number, 2^15 down, of the largest weight
        dl_tol = dl_tol + weight.abs().max() * 2.0 ** -40 if len(keep) else dl_tol
    if dtype != F16:      # a probability below the smallest normal number, 2^-126 in both types, is 0: the exponential and the matrix
        # cores give no smaller one, so dl is off by up to that (float32: so is the third plane of the smallest values)
        dl_tol = dl_tol + weight.abs() * 2.0 ** -126
    dl = dl * weight
    tiny = torch.finfo(dtype).smallest_normal * (1 if dtype != F16 else torch.finfo(dtype).eps)
    dx, dx_tol = torch.zeros((n, d), dtype=torch.float64), torch.zeros((n, d), dtype=torch.float64)
    dx[keep] = dl @ w64
    sums = lambda k: (k + 64) * E  # noqa: E731  (additions of a sum in 32 bits, its splits among them)
    dx_tol[keep] = dl_tol @ w64.abs() + sums(v) * (dl.abs() @ w64.abs()) + (2.0 ** -22 * (dl.abs() @ w64.abs()) if dtype == F32 else 0)
    near(got[0], dx, dx_tol + u * dx.abs() * (1 + 2.0 ** -8) + tiny)
    dw = dl.t() @ xs
    size = dl.abs().t() @ xs.abs()
    near(got[1], dw, dl_tol.t() @ xs.abs() + sums(n) * size + (2.0 ** -22 * size if dtype == F32 else 0) + u * dw.abs() * (1 + 2.0 ** -8) + tiny)
    if b is not None:
        db = dl.sum(0)
        near(got[2], db, dl_tol.sum(0) + sums(n) * dl.abs().sum(0) + u * db.abs() * (1 + 2.0 ** -8) + tiny)
    return loss, got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 2, 8), (3, 20, 64), (127, 129, 67), (128, 128, 64), (129, 20, 96), (257, 260, 128), (500, 33, 30),
                                   (64, 1000, 192), (40, 3001, 16), (2, 700, 513),
                                   (300, 32, 128), (1000, 64, 250), (77, 128, 100), (200, 100, 256), (150, 31, 511), (64, 7, 512), (333, 40, 33), (129, 65, 129), (65, 129, 32), (200, 160, 256),
                                   (64, 200, 255), (1000, 224, 100), (63, 288, 256), (130, 261, 8), (1, 289, 64)])
def test_loss_sizes(pkg, dtype, n, v, d):
    check_loss(pkg, n, v, d, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("bias,target_type,ignore", [(True, torch.int32, 0), (False, torch.int64, -100)])
def test_loss_reductions(pkg, dtype, reduction, bias, target_type, ignore):
    check_loss(pkg, 300, 50, 64, dtype, bias, ignore, reduction, target_type=target_type)
    check_loss(pkg, 300, 150, 64, dtype, bias, ignore, reduction, target_type=target_type)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("piece", [1, 128, 256, 100000])
def test_loss_pieces(pkg, dtype, piece):
    check_loss(pkg, 200, 777, 64, dtype, piece=piece)
    check_loss(pkg, 700, 300, 40, dtype, piece=piece, reduction="none")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_loss_large_logits(pkg, dtype):
    check_loss(pkg, 200, 300, 64, dtype, spread=30.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v,d,share", [(5000, 20, 32, 0.1), (70000, 20, 96, 0.1), (9000, 50, 300, 0.3), (20000, 260, 256, 0.1), (17000, 150, 96, 0.1), (40000, 90, 64, 0.0), (3000, 260, 128, 0.85), (1500, 5000, 64, 0.0), (20, 20000, 128, 0.2)])
def test_loss_larger(pkg, dtype, n, v, d, share):
    check_loss(pkg, n, v, d, dtype, share=share)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,v,d,reduction", [(9000, 1500, 64, "mean"), (2500, 2900, 128, "none"), (70000, 100, 128, "sum"), (33000, 50, 64, "none"),
                                             (600, 40000, 30, "mean"), (7, 30000, 100, "none"), (1, 65, 1, "sum"), (257, 129, 65, "none"), (64, 64, 200, "mean")])
def test_loss_few_features(pkg, dtype, n, v, d, reduction):
    """Logits that are made again: points and classes that end anywhere in what a wave keeps and in what it meets."""
    check_loss(pkg, n, v, d, dtype, reduction=reduction, share=0.15)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v,d", [(33000, 152, 586), (35000, 260, 160), (2000, 5600, 310), (5, 9000, 290), (300, 1100, 512)])
def test_loss_many_features(pkg, dtype, n, v, d):
    check_loss(pkg, n, v, d, dtype, share=0.1)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_loss_where_no_point_counts(pkg, reduction):
    loss, got = check_loss(pkg, 150, 20, 64, BF16, target=torch.full((150,), -100), reduction=reduction)
    assert not loss.any() and not any(t.any() for t in got)


def test_loss_ignored_features_reach_nothing(pkg):
    g = gen(8)
    for dtype, d in ((BF16, 64), (BF16, 50), (F32, 64)):
        x, target = torch.randn((400, d), generator=g).to(dtype), torch.randint(0, 30, (400,), generator=g)
        out = torch.rand((400,), generator=g) < 0.3
        target[out] = -100
        a = check_loss(pkg, 400, 30, d, dtype, x=x, target=target)
        x = x.clone()
        x[out] = float("nan")
        ins = x.cuda().requires_grad_()
        w = (torch.randn((30, d), generator=gen(400 * 7 + 30 * 3 + d)) * 2 / math.sqrt(d)).to(dtype)
        w = w.cuda().requires_grad_()
        loss = pkg.linear_cross_entropy(ins, w, target.cuda(), reduction="sum")
        dx, dw = torch.autograd.grad(loss, (ins, w))
        assert torch.isfinite(loss) and torch.isfinite(dx).all() and torch.isfinite(dw).all() and not dx[out.cuda()].any()
        assert a is not None


def test_loss_masked_classes(pkg):
    """Classes masked by a bias of -inf or the type's lowest value have probability 0; a row that keeps only its own class, loss 0."""
    for dtype in (F32, BF16, F16):
        for low in (float("-inf"), torch.finfo(dtype).min):
            b = torch.zeros(200, dtype=dtype)
            b[50:] = low
            target = torch.arange(90) % 50
            check_loss(pkg, 90, 200, 64, dtype, b=b, target=target)
    b = torch.full((40,), float("-inf"), dtype=BF16)
    b[7] = 0
    loss, got = check_loss(pkg, 30, 40, 64, BF16, b=b, target=torch.full((30,), 7), reduction="none")
    assert loss.abs().max() <= 1e-5 and not got[0].any()
    # the target itself masked: infinite, as the definition says; every class masked: no number
    x, w = torch.randn((3, 64), generator=gen(1)).cuda(), torch.randn((40, 64), generator=gen(2)).cuda()
    loss = pkg.linear_cross_entropy(x, w, torch.tensor([3, 7, 8]).cuda(), bias=b.float().cuda(), reduction="none")
    assert loss[0] == float("inf") and loss[1] == 0 and loss[2] == float("inf")
    loss = pkg.linear_cross_entropy(x, w, torch.tensor([3, 7, 8]).cuda(), bias=torch.full((40,), float("-inf")).cuda(), reduction="none")
    assert torch.isnan(loss).all()


def test_loss_targets_that_are_no_class(pkg):
    x, w = torch.randn((4, 64), generator=gen(1)).cuda().requires_grad_(), torch.randn((20, 64), generator=gen(2)).cuda().requires_grad_()
    loss = pkg.linear_cross_entropy(x, w, torch.tensor([3, 20, -1, 2 ** 40]).cuda(), reduction="none")
    assert torch.isfinite(loss[0]) and torch.isnan(loss[1:]).all()
    dx, = torch.autograd.grad(loss, x, torch.ones(4, device="cuda"))
    assert torch.isfinite(dx[0]).all() and torch.isnan(dx[1:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v,d", [(20, 64), (260, 64), (400, 96)])
def test_loss_infinite_gradients_stay_with_their_points(pkg, dtype, v, d):
    """The gradient of point 3 is infinite, that of point 5 no number: their rows of dx say so, the others are what they are alone."""
    g = gen(v)
    x, w = (torch.randn(s, generator=g).to(dtype).cuda() for s in ((300, d), (v, d)))
    target, up = torch.randint(0, v, (300,), generator=g).cuda(), (torch.rand((300,), generator=g) + 1).cuda() * 40
    target[7] = -100
    bad = up.clone()
    bad[3], bad[5], bad[7], up[3], up[5] = math.inf, math.nan, math.inf, 0, 0

    def dx(u):
        a = x.clone().requires_grad_()
        return torch.autograd.grad(pkg.linear_cross_entropy(a, w, target, reduction="none"), a, u)[0]

    got, want = dx(bad), dx(up)
    assert not torch.isfinite(got[[3, 5]]).any()
    got[[3, 5]] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v,d", [(20, 64), (260, 64), (400, 128), (400, 50)])
def test_loss_tensors_that_were_kept_elsewhere(pkg, dtype, v, d):
    """What the backward pass gets back need not lie as it lay: other strides, other addresses, a single row of any stride."""
    g = gen(v + d)
    x, w, b = (torch.randn(s, generator=g).to(dtype).cuda() for s in ((90, d), (v, d), (v,)))
    target = torch.randint(0, v, (90,), generator=g).cuda()
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()  # noqa: E731

    def moved(t):
        out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return out.copy_(t)

    def wide(t):
        return torch.empty(t.shape[:-1] + (t.shape[-1] + 3,), dtype=t.dtype, device=t.device)[..., :t.shape[-1]].copy_(t)

    def step(x, w, back=None):
        ins = [t.detach().requires_grad_() for t in (x, w, b)]
        if back is None:
            loss = pkg.linear_cross_entropy(ins[0], ins[1], target[:len(x)], bias=ins[2])
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: back(t) if t.is_floating_point() else t):
                loss = pkg.linear_cross_entropy(ins[0], ins[1], target[:len(x)], bias=ins[2])
        return (loss.detach(), *torch.autograd.grad(loss, ins))

    want = step(x, w)
    for back in (turned, moved, wide):
        assert all(torch.equal(p, q) for p, q in zip(step(x, w, back), want))
    one = torch.as_strided(x, (1, d), (1, 1))
    assert all(torch.equal(p, q) for p, q in zip(step(one, w), step(x[:1].clone(), w)))


def test_loss_layouts(pkg):
    g = gen(4)
    for dtype in (BF16, F32):
        base, wide = torch.randn((90, 3, 70), generator=g).to(dtype).cuda(), torch.randn((128, 50), generator=g).to(dtype).cuda()
        target = torch.randint(0, 50, (90, 3), generator=g).cuda()
        for x, w, t in ((base[:, :, 3:67], wide[:64].t(), target), (base[:, 1, :64], wide.t()[:, 10:74], target[:, 1]),
                        (base[:1, :1, :64].expand(90, 3, 64), wide.t()[:, :64], target), (base[0, 0, :64], wide.t()[:, :64], target[0, 0])):
            x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
            loss = pkg.linear_cross_entropy(x, w, t, reduction="sum")
            dx, dw = torch.autograd.grad(loss, (x, w))
            x2, w2 = x.detach().contiguous().requires_grad_(), w.detach().contiguous().requires_grad_()
            l2 = pkg.linear_cross_entropy(x2, w2, t.contiguous(), reduction="sum")
            ex, ew = torch.autograd.grad(l2, (x2, w2))
            assert torch.equal(loss, l2) and torch.equal(dx, ex) and torch.equal(dw, ew) and dx.shape == x.shape
    # a head shared by two losses: the gradients add up
    w = wide.t()[:, :64].detach().contiguous().requires_grad_()
    x = base[:, 0, :64].contiguous()
    one = lambda a, t: torch.autograd.grad(pkg.linear_cross_entropy(a, w, t), w)[0]  # noqa: E731
    both, = torch.autograd.grad(pkg.linear_cross_entropy(x, w, target[:, 0]) + pkg.linear_cross_entropy(x * 2, w, target[:, 1]), w)
    assert torch.equal(both, one(x, target[:, 0]) + one(x * 2, target[:, 1]))


def test_loss_parts_of_the_gradient(pkg):
    g = gen(6)
    x, w, b = torch.randn((70, 64), generator=g).cuda(), torch.randn((30, 64), generator=g).cuda(), torch.randn((30,), generator=g).cuda()
    t = torch.randint(0, 30, (70,), generator=g).cuda()
    ins = [v.clone().requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(pkg.linear_cross_entropy(ins[0], ins[1], t, bias=ins[2]), ins)
    for k in range(3):
        some = [v.clone().requires_grad_(i == k) for i, v in enumerate((x, w, b))]
        got, = torch.autograd.grad(pkg.linear_cross_entropy(some[0], some[1], t, bias=some[2]), some[k])
        assert torch.equal(got, want[k])
    assert not pkg.linear_cross_entropy(x, w, t).requires_grad
    # backward twice through one forward
    loss = pkg.linear_cross_entropy(ins[0], ins[1], t, bias=ins[2])
    for _ in range(2):
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(loss, ins, retain_graph=True), want))


def test_second_derivatives_are_refused(pkg):
    x, w = torch.randn((40, 64), generator=gen(1)).cuda().requires_grad_(), torch.randn((30, 64), generator=gen(2)).cuda().requires_grad_()
    t = torch.randint(0, 30, (40,), generator=gen(3)).cuda()
    plain, = torch.autograd.grad(pkg.linear_cross_entropy(x, w, t), x)
    dx, = torch.autograd.grad(pkg.linear_cross_entropy(x, w, t), x, create_graph=True)      # (harmless as long as nobody follows it)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError, match="once"):
        (dx ** 2).sum().backward()
    q, pos = torch.randn((40, 2, 8), generator=gen(4)).cuda().requires_grad_(), torch.randn((40, 1), generator=gen(5)).cuda()
    dq, = torch.autograd.grad((pkg.rotary_positions(q, pos, (4,))[0] ** 3).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        dq.sum().backward()


def test_loss_of_no_points(pkg):
    w = torch.randn((30, 64), device="cuda").requires_grad_()
    x = torch.zeros((0, 64), device="cuda").requires_grad_()
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    for reduction, shape in (("mean", ()), ("sum", ()), ("none", (0,))):
        loss = pkg.linear_cross_entropy(x, w, t, reduction=reduction)
        assert loss.shape == shape and not loss.any()
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert dx.shape == (0, 64) and not dw.any()


def test_loss_gradient_against_differences(pkg):
    g = gen(9)
    x, w, b = (torch.randn(s, generator=g).cuda().requires_grad_() for s in ((12, 16), (9, 16), (9,)))
    t = torch.randint(0, 9, (12,), generator=g).cuda()
    f = lambda *a: pkg.linear_cross_entropy(a[0], a[1], t, bias=a[2], reduction="sum").item()  # noqa: E731
    got = torch.autograd.grad(pkg.linear_cross_entropy(x, w, t, bias=b, reduction="sum"), (x, w, b))
    h = 2.0 ** -6
    for k, at in ((0, (3, 5)), (0, (11, 15)), (1, (0, 0)), (1, (8, 7)), (2, (4,))):
        up, down = [v.detach().clone() for v in (x, w, b)], [v.detach().clone() for v in (x, w, b)]
        up[k][at] += h
        down[k][at] -= h
        # third derivative of the loss below 30 (|w|, |x| < 4) times h^2 / 6; the sum's rounding over 2 h
        assert abs(got[k][at].item() - (f(*up) - f(*down)) / (2 * h)) <= 30 * h * h / 6 + 200 * E / h


def test_operators_on_another_stream_and_in_a_graph(pkg):
    g = gen(11)
    q = torch.randn((260, 2, 32), generator=g).to(BF16).cuda()
    pos = torch.randn((260, 3), generator=g).cuda() * 9
    w = torch.randn((21, 64), generator=g).to(BF16).cuda()
    t = torch.randint(0, 21, (260,), generator=g).cuda()

    def step(q, w):
        y, _ = pkg.rotary_positions(q, pos, (5, 5, 5))
        loss = pkg.linear_cross_entropy(y.flatten(1), w, t, ignore_index=0)
        return (loss, *torch.autograd.grad(loss, (q, w)))

    def eager(q, w):
        return [v.detach().clone() for v in step(q.detach().clone().requires_grad_(), w.detach().clone().requires_grad_())]

    want = eager(q, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eager(q, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs of the same step over leaves of their own, replayed in turn with new values and eager work between
    graphs = []
    for _ in range(2):
        a, b = q.clone().requires_grad_(), w.clone().requires_grad_()
        with torch.cuda.stream(side):
            step(a, b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(a, b)
        graphs.append((graph, a, b, out))
    for k in range(4):
        for graph, a, b, out in graphs:
            with torch.no_grad():
                a.copy_(torch.randn(q.shape, generator=g).to(BF16))
                b.copy_(torch.randn(w.shape, generator=g).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager(a, b))), k


@pytest.mark.parametrize("dtype,v,d,reduction", [(BF16, 260, 64, "none"), (F16, 260, 128, "none"), (BF16, 400, 96, "mean"), (F32, 400, 64, "sum"), (F32, 50, 64, "none")])
def test_loss_of_many_classes_in_a_graph(pkg, dtype, v, d, reduction):
    """Forward and backward of every way the head is taken, captured; replayed with new points, labels and gradients."""
    g = gen(v)
    n = 700
    x, w, up = torch.randn((n, d), generator=g).to(dtype).cuda(), torch.randn((v, d), generator=g).to(dtype).cuda(), torch.rand((n,), generator=g).cuda()
    b, target = torch.randn((v,), generator=g).to(dtype).cuda(), torch.randint(-1, v, (n,), generator=g).cuda()

    def step(x, w, b):
        loss = pkg.linear_cross_entropy(x, w, target, bias=b, ignore_index=-1, reduction=reduction)
        return (loss, *torch.autograd.grad(loss, (x, w, b), up if reduction == "none" else up[0]))

    def eager():
        return [t.detach().clone() for t in step(*(t.detach().clone().requires_grad_() for t in (x, w, b)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    with torch.cuda.stream(side):
        step(*leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves)
    for k in range(4):
        share = (0.0, 0.3, 1.0, 0.9)[k]
        x.normal_()
        up.uniform_(-1, 1)
        target.copy_(torch.where(torch.rand((n,), generator=g) < share, -1, torch.randint(0, v, (n,), generator=g)))
        with torch.no_grad():
            leaves[0].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager())), k


def test_two_losses_at_once_on_two_streams(pkg):
    g = gen(12)
    work = []
    for v, d, n, dtype in ((20, 96, 60000, BF16), (260, 128, 30000, F16), (700, 64, 20000, BF16), (30, 64, 20000, F32)):
        x, w = (torch.randn(s, generator=g).to(dtype).cuda().requires_grad_() for s in ((n, d), (v, d)))
        work.append((x, w, torch.randint(-1, v, (n,), generator=g).cuda()))

    def step(x, w, t):
        loss = pkg.linear_cross_entropy(x, w, t, ignore_index=-1)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    want = [step(*p) for p in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for turn in range(3):
        got = []
        for s, p in zip(streams, work[turn:] + work[:turn]):
            with torch.cuda.stream(s):
                got.append(step(*p))
        torch.cuda.synchronize()
        for a, b in zip(got, want[turn:] + want[:turn]):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---- beyond 32 bits ------------------------------------------------------------------------------------------------------------
def test_rotary_beyond_32_bits(pkg):
    tokens, heads, dim = 4_300_001, 8, 64      # 2.2e9 elements
    q = torch.empty((tokens, heads, dim), dtype=BF16, device="cuda").normal_()
    pos = torch.empty((tokens, 3), device="cuda").uniform_(-50, 50)
    y, _ = pkg.rotary_positions(q, pos, (10, 10, 10))
    at = torch.tensor([0, 1, 2 ** 21, 4_194_303, 4_194_304, 4_194_305, tokens - 2, tokens - 1])
    near(y[at.cuda()], *rotate64(q[at.cuda()], pos[at.cuda()], (10, 10, 10), 10000.0, "half"))


@pytest.mark.parametrize("n,v,d", [(9_000_001, 20, 256), (8_500_001, 200, 256), (4_300_001, 300, 512)])
def test_loss_beyond_32_bits(pkg, n, v, d):
    """More than 2^31 features: loss and dx at points along the way, db of all (against the definition in 32 bits, in parts)."""
    x = torch.empty((n, d), dtype=BF16, device="cuda").normal_().requires_grad_()
    w = (torch.randn((v, d), generator=gen(v)) / math.sqrt(d)).to(BF16).cuda().requires_grad_()
    b = torch.zeros((v,), dtype=BF16, device="cuda").requires_grad_()
    target = torch.randint(0, v, (n,), device="cuda")
    target[torch.rand((n,), device="cuda") < 0.1] = -100
    loss = pkg.linear_cross_entropy(x, w, target, bias=b, reduction="none")
    up = torch.rand((n,), device="cuda")
    dx, dw, db = torch.autograd.grad(loss, (x, w, b), up)
    at = torch.cat([torch.arange(0, n, n // 200, device="cuda"), torch.tensor([n - 1, 2 ** 31 // d, 2 ** 31 // d - 1, 2 ** 32 // d - 1], device="cuda").clamp(max=n - 1)])
    x64, w64, t = x.detach()[at].double().cpu(), w.detach().double().cpu(), target[at].cpu()
    keep = (t != -100).double()
    logits = x64 @ w64.t()
    lse = torch.logsumexp(logits, 1)
    each = (lse - logits[torch.arange(len(at)), t.clamp(min=0)]) * keep
    e_l = (d + 16) * E * ((x64.abs() @ w64.abs().t()).amax(1) + 1)
    near(loss[at], each, 2 * e_l + 8 * E * (lse.abs() + each.abs()))
    dl = torch.exp(logits - lse[:, None])
    p = dl.clone()
    dl[torch.arange(len(at)), t.clamp(min=0)] -= 1
    by = (up[at].double().cpu() * keep)[:, None]
    tol = (p * (2 * e_l[:, None] + 2.0 ** -20) + 2.0 ** -8 * dl.abs()) * by + 2.0 ** -126
    size = (dl * by).abs() @ w64.abs()
    near(dx[at], (dl * by) @ w64, (tol @ w64.abs() + (v + 64) * E * size) * (1 + 2.0 ** -8) + 2.0 ** -8 * ((dl * by) @ w64).abs() + 2.0 ** -126)
    want, total = torch.zeros((v,), dtype=torch.float64, device="cuda"), torch.zeros((v,), dtype=torch.float64, device="cuda")
    want_w, total_w = torch.zeros((v, d), dtype=torch.float64, device="cuda"), torch.zeros((v, d), dtype=torch.float64, device="cuda")
    for part in range(0, n, 200_000):
        xs, ts, us = x.detach()[part:part + 200_000].double(), target[part:part + 200_000], up[part:part + 200_000].double()
        g = torch.softmax(xs @ w.detach().double().t(), 1)
        g[torch.arange(len(ts), device="cuda"), ts.clamp(min=0)] -= 1
        g *= (us * (ts != -100))[:, None]
        want += g.sum(0)
        total += g.abs().sum(0)
        want_w += g.t().contiguous() @ xs
        total_w += g.abs().t().contiguous() @ xs.abs()
    # a probability is off by 2 e_l + 2^-20 of itself, dl of dW by half a step of bfloat16; additions in 32 bits, in chains of at
    # most 2^14 (a chain's rounding is off by its length times E of what it has summed)
    rel = 2 * float(e_l.max()) * 2 + 2.0 ** -20 + 2.0 ** 14 * E
    assert ((db.double() - want).abs() <= rel * total + 2.0 ** -8 * want.abs()).all()
    assert ((dw.double() - want_w).abs() <= (rel + 2.0 ** -8) * total_w + 2.0 ** -8 * want_w.abs()).all()


WAYS = [(20, 64, BF16), (50, 100, F32), (400, 64, F16), (300, 100, F32), (1000, 128, BF16), (150, 192, F16), (288, 128, BF16), (400, 160, BF16), (150, 190, F32)]


@pytest.mark.parametrize("v,d,dtype", WAYS)
def test_loss_masked_and_large_every_way(pkg, v, d, dtype):
    """Masked classes (-inf, the lowest value), logits up to +-300, targets that are masked, no class or not counted, rows of NaN that
    do not count -- in every way a head is taken."""
    g = gen(v * d)
    n = 230
    target = torch.arange(n) % (v // 2)
    for low in (float("-inf"), torch.finfo(dtype).min):
        b = torch.randn((v,), generator=g).to(dtype)
        b[v // 2:] = low
        check_loss(pkg, n, v, d, dtype, b=b, target=target, seed=3)
    x = torch.randn((n, d), generator=g).to(dtype)
    w = torch.randn((v, d), generator=g).to(dtype)
    w[::7] *= 100 / math.sqrt(d)
    check_loss(pkg, n, v, d, dtype, x=x, w=w, target=torch.randint(0, v, (n,), generator=g), reduction="none")
    # what is not finite stays where it is
    b = torch.zeros((v,), dtype=dtype)
    b[5] = float("-inf")
    odd = torch.randint(6, v, (n,), generator=g)
    odd[3], odd[40], odd[100], odd[229] = 5, v, -7, -100
    x[229] = float("nan")
    x[41] = float("inf")
    xg, wg = x.cuda().requires_grad_(), (w * 0.01).to(dtype).cuda()
    loss = pkg.linear_cross_entropy(xg, wg, odd.cuda(), bias=b.cuda(), reduction="none")
    assert loss[3] == float("inf") and torch.isnan(loss[[40, 41, 100]]).all() and loss[229] == 0
    rest = torch.ones(n, dtype=torch.bool)
    rest[[3, 40, 41, 100]] = False
    assert torch.isfinite(loss[rest.cuda()]).all()
    dx, = torch.autograd.grad(loss, xg, torch.ones(n, device="cuda"))
    rest[3] = True      # (its probability is 0: a gradient like any other)
    assert torch.isfinite(dx[rest.cuda()]).all() and torch.isnan(dx[[40, 41, 100]]).all() and not dx[229].any()
    b[:] = float("-inf")
    assert torch.isnan(pkg.linear_cross_entropy(xg[:3], wg, odd[:3].cuda(), bias=b.cuda(), reduction="none")).all()


@pytest.mark.parametrize("v,d,dtype", WAYS)
def test_loss_repeats_its_bits_every_way(pkg, v, d, dtype):
    """The same inputs give the same bits, beside other work, and with points that do not count in between."""
    g = gen(v + d)
    n = 3001
    x, w, b = (torch.randn(s, generator=g).to(dtype).cuda().requires_grad_() for s in ((n, d), (v, d), (v,)))
    target = torch.randint(-3, v, (n,), generator=g).clamp(min=-1).cuda()

    def step(reduction):
        loss = pkg.linear_cross_entropy(x, w, target, bias=b, ignore_index=-1, reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss.sum(), (x, w, b)))

    for reduction in ("mean", "none"):
        want = step(reduction)
        noise = torch.randn((2000, 2000), device="cuda")
        for _ in range(4):
            noise = noise @ noise * 1e-3
            assert all(torch.equal(p, q) for p, q in zip(step(reduction), want))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_loss_of_no_points_whatever_the_head_holds(pkg, dtype):
    w = torch.ones((2000, 64), dtype=dtype, device="cuda")
    b = torch.zeros(2000, dtype=dtype, device="cuda")
    w[3, 5], b[7] = float("inf"), float("-inf")
    for head, bias in ((w, b), (torch.ones_like(w), None), (torch.full_like(w, torch.finfo(dtype).max), b)):
        ins = [t.clone().requires_grad_() for t in (torch.zeros((0, 64), dtype=dtype, device="cuda"), head) + (() if bias is None else (bias,))]
        for reduction in ("mean", "sum", "none"):
            loss = pkg.linear_cross_entropy(ins[0], ins[1], torch.zeros(0, dtype=torch.int64, device="cuda"), bias=None if bias is None else ins[2], reduction=reduction)
            assert loss.dtype == F32 and loss.shape == ((0,) if reduction == "none" else ()) and (loss == 0).all()
            got = torch.autograd.grad(loss.sum(), ins)
            assert all(g.shape == t.shape and g.dtype == dtype and not g.any() for g, t in zip(got, ins))


FEW = [(20, 64, F16), (20, 64, F32), (100, 96, BF16), (40, 200, F16)]      # flavours of the few classes' way that WAYS leaves out


@pytest.mark.parametrize("v,d,dtype", WAYS + FEW)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_loss_points_that_do_not_count_have_no_gradient_whatever_comes_in(pkg, v, d, dtype, reduction):
    g = gen(v + d)
    n = 301
    x, w = (torch.randn(s, generator=g).to(dtype).cuda().requires_grad_() for s in ((n, d), (v, d)))
    target = torch.randint(0, v, (n,), generator=g)
    out = torch.rand((n,), generator=g) < 0.4
    target[out] = -100
    loss = pkg.linear_cross_entropy(x, w, target.cuda(), reduction=reduction)
    for up in (math.inf, -math.inf, math.nan):
        dx, = torch.autograd.grad(loss, x, torch.tensor(up).cuda(), retain_graph=True)
        assert (dx[out.cuda()] == 0).all() and not torch.isfinite(dx[~out.cuda()]).any()


@pytest.mark.parametrize("v,d,dtype", WAYS + FEW)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_without_points_that_count_has_no_gradient_whatever_comes_in(pkg, v, d, dtype, reduction):
    g = gen(v + d)
    n = 150
    ins = [torch.randn(s, generator=g).to(dtype).cuda().requires_grad_() for s in ((n, d), (v, d), (v,))]
    loss = pkg.linear_cross_entropy(ins[0], ins[1], torch.full((n,), -100).cuda(), bias=ins[2], reduction=reduction)
    for up in (math.inf, math.nan):
        got = torch.autograd.grad(loss, ins, torch.full(loss.shape, up, device="cuda"), retain_graph=True)
        assert all((t == 0).all() for t in got)


def test_rotary_refuses_forward_mode(pkg):
    q, k, pos = torch.randn((5, 2, 8)).cuda(), torch.randn((5, 1, 8)).cuda(), torch.randn((5, 1)).cuda()
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for a, p, b in ((dual(q), pos, k), (q, pos, dual(k)), (q, dual(pos), k), (dual(q), pos, None)):
            with pytest.raises(RuntimeError):
                pkg.rotary_positions(a, p, (4,), key=b)
            with torch.no_grad(), pytest.raises(RuntimeError):
                pkg.rotary_positions(a, p, (4,), key=b)
        plain = pkg.rotary_positions(q, pos, (4,), key=k)
    want = pkg.rotary_positions(q, pos, (4,), key=k)
    assert all(torch.equal(a, b) for a, b in zip(plain, want))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: pkg.rotary_positions(t, pos, (4,))[0], (q,), (q,))


def test_loss_refuses_forward_mode(pkg):
    x, w, t = torch.randn((5, 8)).cuda(), torch.randn((3, 8)).cuda(), torch.zeros(5, dtype=torch.int64).cuda()
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError):
            pkg.linear_cross_entropy(dual, w, t)
        with torch.no_grad(), pytest.raises(RuntimeError):
            pkg.linear_cross_entropy(dual, w, t)
        wd = fwd.make_dual(w, torch.ones_like(w))
        with pytest.raises(RuntimeError):
            pkg.linear_cross_entropy(x, wd, t)


def test_gradients_refuse_forward_mode(pkg):
    q, pos = torch.randn((5, 2, 8)).cuda().requires_grad_(), torch.randn((5, 1)).cuda()
    x, w, t = torch.randn((5, 8)).cuda().requires_grad_(), torch.randn((3, 8)).cuda(), torch.zeros(5, dtype=torch.int64).cuda()
    y, loss = pkg.rotary_positions(q, pos, (4,))[0], pkg.linear_cross_entropy(x, w, t)
    with fwd.dual_level():
        for out, leaf in ((y, q), (loss, x)):
            up = torch.ones_like(out).detach()
            want, = torch.autograd.grad(out, leaf, up, retain_graph=True)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaf, fwd.make_dual(up, torch.ones_like(up)), retain_graph=True)
            assert torch.equal(torch.autograd.grad(out, leaf, up, retain_graph=True)[0], want)


def test_tensors_that_are_negated_when_they_are_read(pkg):
    """Views with the bit that torch resolves at the next read: refused as inputs, right as gradients."""
    minus = torch._neg_view
    q, pos = torch.randn((5, 2, 8)).cuda(), torch.randn((5, 1)).cuda()
    x, w, t = torch.randn((5, 8)).cuda(), torch.randn((3, 8)).cuda(), torch.zeros(5, dtype=torch.int64).cuda()
    rows, s = torch.randn((5, 4), dtype=torch.complex64).cuda(), torch.tensor([1, 0]).cuda()
    for call in (lambda: pkg.rotary_positions(minus(q), pos, (4,)), lambda: pkg.rotary_positions(q, minus(pos), (4,)),
                 lambda: pkg.rotary_positions(q, pos, (4,), key=minus(q)), lambda: pkg.linear_cross_entropy(minus(x), w, t),
                 lambda: pkg.linear_cross_entropy(x, minus(w), t), lambda: pkg.linear_cross_entropy(x, w, t, bias=minus(w[:, 0].contiguous())),
                 lambda: pkg.take_rows(s, (rows.conj(),)), lambda: pkg.put_rows(s, (rows[:2],), (rows.conj(),)),
                 lambda: pkg.take_rows(s, (minus(x),)), lambda: pkg.put_rows(s, (minus(x),), (x.clone(),))):
        with pytest.raises(ValueError, match="resolve"):
            call()
    assert torch.equal(pkg.take_rows(s, (rows.conj().resolve_conj(),))[0], rows.conj()[s])
    q.requires_grad_()
    x.requires_grad_()
    for out, leaf in ((pkg.rotary_positions(q, pos, (4,))[0], q), (pkg.linear_cross_entropy(x, w, t, reduction="none"), x)):
        up = torch.randn(out.shape).cuda()
        one, two = (torch.autograd.grad(out, leaf, g, retain_graph=True)[0] for g in (minus(up), -up))
        assert torch.equal(one, two)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotary_positions_that_were_kept_elsewhere(pkg, dtype):
    g = gen(3)
    pos = torch.randn((40, 4), generator=g).cuda() * 20
    up = torch.randn((40, 3, 24), generator=g).to(dtype).cuda()

    def step(back=None):
        q = torch.ones((40, 3, 24), dtype=dtype, device="cuda", requires_grad=True)
        if back is None:
            y, _ = pkg.rotary_positions(q, pos[:, :3], (4, 4, 3))
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
                y, _ = pkg.rotary_positions(q, pos[:, :3], (4, 4, 3))
        return torch.autograd.grad(y, q, up)[0]

    want = step()
    for back in (lambda t: t.t().contiguous().t(), lambda t: t.clone(), lambda t: t.cpu().cuda()):
        assert torch.equal(step(back), want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,v,d", [(3001, 260, 128), (2500, 150, 192), (1030, 288, 96), (700, 130, 256)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_of_a_head_in_lds_by_points(pkg, dtype, n, v, d, reduction):
    """Heads whose points are cut so that the gradients of `piece` classes are held at a time: the same as without, but for the order
    in which dweight is added up; dx of a point does not depend on it."""
    whole = check_loss(pkg, n, v, d, dtype, reduction=reduction, share=0.3)
    for piece in (1, 128, 192):
        loss, got = check_loss(pkg, n, v, d, dtype, reduction=reduction, share=0.3, piece=piece)
        assert torch.equal(loss, whole[0]) and torch.equal(got[0], whole[1][0])


def test_loss_of_a_head_in_lds_by_points_where_some_parts_count_nothing(pkg):
    """The points that count are in front of the line: the launches behind have none."""
    g = gen(2)
    n, v, d = 4000, 260, 128
    for counted in (0, 1, 256, 700):
        target = torch.full((n,), -100)
        target[torch.randperm(n, generator=g)[:counted]] = torch.randint(0, v, (counted,), generator=g)
        check_loss(pkg, n, v, d, BF16, target=target, piece=64)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("piece", [1, 128, 192, 256, 100000])
@pytest.mark.parametrize("n,v,d", [(200, 777, 160), (700, 900, 200), (300, 641, 130)])
def test_loss_pieces_of_many_classes(pkg, dtype, piece, n, v, d):
    """Heads whose gradients go through memory a piece of the classes at a time (more than 288 classes and 128 features): sums
    that go on from piece to piece, pieces that end inside a tile, a short last one."""
    for reduction in ("none", "mean"):
        loss, got = check_loss(pkg, n, v, d, dtype, reduction=reduction, piece=piece)
        again = check_loss(pkg, n, v, d, dtype, reduction=reduction, piece=piece)
        assert torch.equal(loss, again[0]) and all(torch.equal(a, b) for a, b in zip(got, again[1]))


@pytest.mark.parametrize("v,d,dtype", WAYS + FEW)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_parts_of_the_gradient_every_way(pkg, v, d, dtype, reduction):
    """The gradient of one of features, head and bias alone, of two, and the loss without any, also in inference mode."""
    g = gen(v * 3 + d)
    n = 400
    ins = [torch.randn(s, generator=g).to(dtype).cuda() for s in ((n, d), (v, d), (v,))]
    target, up = torch.randint(-1, v, (n,), generator=g).cuda(), torch.rand((n,), generator=g).cuda()

    def step(need):
        some = [t.clone().requires_grad_(k in need) for k, t in enumerate(ins)]
        loss = pkg.linear_cross_entropy(some[0], some[1], target, bias=some[2], ignore_index=-1, reduction=reduction)
        return loss, torch.autograd.grad(loss, [some[k] for k in need], up if reduction == "none" else up[0])

    loss, want = step((0, 1, 2))
    for need in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        one, got = step(need)
        assert torch.equal(one, loss) and all(torch.equal(got[i], want[k]) for i, k in enumerate(need)), need
    with torch.inference_mode():
        assert torch.equal(pkg.linear_cross_entropy(ins[0], ins[1], target, bias=ins[2], ignore_index=-1, reduction=reduction), loss)


@pytest.mark.parametrize("v,d,dtype", WAYS + FEW)
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_loss_of_a_head_that_is_sure_of_itself(pkg, v, d, dtype, reduction):
    """Large logits, one class ahead of its only rival by 8: the loss is 3e-4 beside a maximum of some 200 to 300, and so are the
    gradients.  Logits are whole numbers and exact; in units of log 2 (t, at most T) they are rounded, off by E T each, so the rival's part is off
    by rho = ln 2 (2 E T + 2 E |t - top|) + 2^-22 of itself, whatever the rest of the way.  Sum and target's gradient: 4 additions to a
    number near 1 (all other parts are below 2^-30: together below a step), E each."""
    g = gen(v + d)
    n = 300
    w = (torch.randint(0, 2, (v, d), generator=g) * 2 - 1).double()
    w[:, 0] = 1
    w[1::2] = w[::2]
    w[1::2, 1:5] *= -1      # a class's rival differs in four features
    target = torch.randint(0, v, (n,), generator=g)
    x = w[target].clone()
    x[:, 0] = 128
    logits = x @ w.t()
    gap = (logits.amax(1, keepdim=True) - logits).sort(1).values
    assert (gap[:, 0] == 0).all() and (gap[:, 1] == 8).all() and (gap[:, 2] > 21).all()
    up = torch.rand((n,), generator=g) + 0.5 if reduction == "none" else torch.tensor(1.5)
    ins = [t.to(dtype).cuda().requires_grad_() for t in (x, w, torch.zeros(v))]
    loss = pkg.linear_cross_entropy(ins[0], ins[1], target.cuda(), bias=ins[2], reduction=reduction)
    dx, dw, db = torch.autograd.grad(loss, ins, up.cuda())
    large = logits.abs().amax(1, keepdim=True) * 1.4427
    rho = math.log(2) * (2 * E * large + 2 * E * 12) + 2.0 ** -22
    p = torch.softmax(logits, 1)
    rest = p.scatter(1, target[:, None], 0).sum(1, keepdim=True)      # 1 - p of the target, without the subtraction
    each = torch.log1p(rest / (1 - rest))
    each_tol = rho * rest + 8 * E + 4 * E * each
    if reduction == "none":
        near(loss, each[:, 0], each_tol[:, 0])
    else:
        near(loss, each.sum(), each_tol.sum())
    u = torch.finfo(dtype).eps / 2
    dl = p.scatter(1, target[:, None], -rest)
    tol = (rho + 8 * E + (2.0 ** -22 if dtype == F32 else u)) * dl.abs()
    tol = tol.scatter_add(1, target[:, None], torch.full((n, 1), 8 * E, dtype=torch.float64))
    weight = up.double().expand(n)[:, None]
    dl, tol = dl * weight, tol * weight
    tol = tol + weight.max() * (2.0 ** -40 if dtype == F16 else 2.0 ** -126)
    for got, a, b, terms in ((dx, dl, w, v), (dw, dl.t(), x, n), (db, dl.t(), torch.ones((n, 1), dtype=torch.float64), n)):
        want, size = a @ b, a.abs() @ b.abs()
        bound = (tol if a is dl else tol.t()) @ b.abs() + ((terms + 64) * E + (2.0 ** -22 if dtype == F32 else 0)) * size + u * want.abs() * (1 + 2.0 ** -8) + torch.finfo(dtype).smallest_normal
        near(got.reshape(want.shape), want, bound)


@pytest.mark.parametrize("v,d,dtype", [w for w in WAYS + FEW if w[2] != F16])
def test_loss_of_a_bias_past_the_range(pkg, v, d, dtype):
    """The lowest float32 and bfloat16 are past the range in units of log 2: they mask a class as -inf does, its own points included."""
    g = gen(v)
    x, w = (torch.randn(s, generator=g).to(dtype).cuda() for s in ((90, d), (v, d)))
    target = torch.arange(90).cuda() % v
    for low in (torch.finfo(dtype).min, -2.5e38):
        b, c = torch.zeros((v,), dtype=dtype, device="cuda"), torch.zeros((v,), dtype=dtype, device="cuda")
        b[::3], c[::3] = low, -math.inf
        got, want = (pkg.linear_cross_entropy(x, w, target, bias=t, reduction="none") for t in (b, c))
        assert torch.equal(got, want) and torch.isinf(got[target % 3 == 0]).all() and torch.isfinite(got[target % 3 != 0]).all()
