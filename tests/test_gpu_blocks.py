"""GPU tests of the conditioned image block's operators (blocks.py) against
their definitions in 64 bits, which stand here.

Bounds, element by element. u is the unit roundoff of the element type (2^-24,
2^-11, 2^-8). A result is rounded once: u |exact|. Sums of products are float32
in a fixed order: at most 64 roundings' worth (the square root of the longest
sum here, and the score's own rounding inside exp) of the sum of the
products' absolute values. Where 16-bit operands go through the tensor cores,
the probabilities and score gradients are rounded to the element type too:
2 u of that sum (their own rounding, and the one of the output that delta is
taken from). float16 adds half its smallest step, 2^-25."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def rdv():
    import rdv_project_b200 as rdv

    yield rdv
    assert rdv.device_status() == 0


def near(got, exact, dtype, mass, operand_roundings=2):
    """got within the bound of exact; mass: the sum of the absolute values of
    the products behind each element."""
    u = U[dtype]
    operands = 0.0 if dtype == torch.float32 else operand_roundings * u
    bound = u * exact.abs() + (operands + 64 * 2.0 ** -24) * mass + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (got.double() - exact).abs()
    assert got.shape == exact.shape and torch.isfinite(got).all()
    worst = (off / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, worst


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------- group norm


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    return z


def norm64(x, groups, w, b, eps, act):
    n, c = x.shape[0], x.shape[-1]
    xs = x.reshape(n, -1, groups, c // groups)
    mean = xs.mean((1, 3), keepdim=True)
    var = ((xs - mean) ** 2).mean((1, 3), keepdim=True)
    hat = ((xs - mean) / (var + eps).sqrt()).reshape(x.shape)
    return act64(hat * (1 if w is None else w) + (0 if b is None else b), act)


NORM_SHAPES = [((1, 1, 4), 2), ((2, 3, 5, 6), 3), ((3, 37, 53, 60), 6), ((1, 16, 16, 64), 8), ((2, 100, 2056), 8),
               ((5, 7, 33), 11), ((2, 9, 33), 33), ((3, 64, 8, 512), 32), ((1, 5000, 8), 1), ((40, 4, 24), 24),
               ((1, 3, 4100), 4), ((2, 300, 31, 2), 1), ((1, 70001, 16), 4)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", NORM_SHAPES)
def test_group_norm_forward_and_gradients(rdv, cuda_device, dtype, shape, groups):
    g = gen(len(shape) * 100 + groups)
    act = [None, "relu", "silu", "gelu"][(groups + shape[1]) % 4]
    c = shape[-1]
    x = randn(g, *shape, dtype=dtype, scale=1.5)
    x = (x + randn(g, c)).to(dtype)
    w, b = 1 + 0.2 * randn(g, c), 0.2 * randn(g, c)
    dy = randn(g, *shape, dtype=dtype, scale=0.1)
    xd, wd, bd = (t.double().requires_grad_() for t in (x, w, b))
    yd = norm64(xd, groups, wd, bd, 1e-5, act)
    yd.backward(dy.double())
    y, stats = rdv.group_norm_forward(x, groups, w, b, activation=act)
    assert torch.equal(y, rdv.group_norm(x, groups, w, b, activation=act))
    # a normalised value carries the mean's rounding: as many of its own as the mean has deviations
    n = shape[0]
    xs = x.double().reshape(n, -1, groups, c // groups)
    dev = (xs.var((1, 3), unbiased=False) + 1e-5).sqrt()
    far = 1 + (xs.mean((1, 3)).abs() / dev).amax().item()
    hat = norm64(x.double(), groups, None, None, 1e-5, None)
    near(y, yd.detach(), dtype, far + hat.abs() * w.abs() + b.abs(), operand_roundings=0)
    near(stats[..., 0].double(), xs.mean((1, 3)), torch.float32, xs.abs().mean((1, 3)))
    near(stats[..., 1].double(), 1 / dev, torch.float32, far / dev)
    dx, dw, db = rdv.group_norm_backward(dy, x, stats, groups, w, b, activation=act)
    slope = 1.2  # the largest derivative of the activations
    reach = dy.double().abs().amax() * slope * w.double().abs().amax() * far
    near(dx, xd.grad, dtype, (reach * (1 + hat.abs()) ** 2).reshape(xs.shape).div(dev[:, None, :, None])
         .reshape(x.shape), operand_roundings=0)
    pos = tuple(range(len(shape) - 1))
    # relu's derivative jumps where a rounding moves z across 0: one element there
    jump = dy.double().abs().amax() * (1 + hat.abs().amax()) * 2.0 ** 24 / 64 if act == "relu" else 0.0
    crossing = ((hat * w + b).abs() < 1e-5).any() if act == "relu" else False
    extra = jump if crossing else 0.0
    near(dw, wd.grad, torch.float32, far * slope * (dy.double().abs() * (1 + hat.abs())).sum(pos) + extra)
    near(db, bd.grad, torch.float32, far * slope * dy.double().abs().sum(pos) + extra)


def test_group_norm_far_mean_and_strides(rdv, cuda_device):
    g = gen(5)
    x = randn(g, 2, 40, 24, 64) + 3000.0  # 3000 deviations from 0
    exact = norm64(x.double(), 8, None, None, 1e-5, None)
    # the mean in float32 is off by at most half its step, 2^-13, of a deviation of 1
    assert (rdv.group_norm(x, 8).double() - exact).abs().max() < 2.0 ** -13 + 64 * 2.0 ** -24 * 6
    wide = randn(g, 2, 40, 24, 128, dtype=torch.float16)
    part = wide[..., 3:67]  # another stride and an odd offset
    assert torch.equal(rdv.group_norm(part, 8, activation="silu"),
                       rdv.group_norm(part.contiguous(), 8, activation="silu"))
    flat = randn(g, 2 * 40 * 64 + 1, dtype=torch.bfloat16)
    odd = flat[1:].view(2, 40, 64)  # dense, off the 16-byte grid
    near(rdv.group_norm(odd, 4), norm64(odd.double(), 4, None, None, 1e-5, None), torch.bfloat16,
         1 + norm64(odd.double(), 4, None, None, 1e-5, None).abs(), 0)
    half = randn(g, 64, dtype=torch.float16)
    both = rdv.group_norm(odd, 4, half, half)
    assert torch.equal(both, rdv.group_norm(odd, 4, half.float(), half.float()))
    assert torch.equal(rdv.group_norm(odd, 4, half, None), rdv.group_norm(odd, 4, half.float(), torch.zeros_like(half)))


def test_group_norm_constant_empty_and_nan(rdv, cuda_device):
    y, stats = rdv.group_norm_forward(torch.full((2, 9, 8), 7.0, device=cuda_device), 2)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(stats[..., 0], torch.full_like(stats[..., 0], 7.0))
    assert rdv.group_norm(torch.zeros(0, 9, 8, device=cuda_device), 2).shape == (0, 9, 8)
    x = torch.zeros(2, 0, 8, device=cuda_device)
    y, stats = rdv.group_norm_forward(x, 2)
    dx, dw, db = rdv.group_norm_backward(y, x, stats, 2, torch.ones(8), torch.ones(8))
    assert dx.shape == x.shape and not dw.any() and not db.any()
    x = randn(gen(1), 2, 50, 8)
    x[0, 3, 1] = math.nan
    y = rdv.group_norm(x, 2, activation="relu")
    assert torch.isnan(y[0, :, :4]).all() and torch.isfinite(y[0, :, 4:]).all() and torch.isfinite(y[1]).all()


def test_group_norm_repeats_and_differences(rdv, cuda_device):
    g = gen(9)
    x, w, b, dy = randn(g, 3, 33, 17, 48), 1 + 0.2 * randn(g, 48), 0.2 * randn(g, 48), randn(g, 3, 33, 17, 48)
    for act in (None, "silu", "gelu"):
        y, stats = rdv.group_norm_forward(x, 6, w, b, activation=act)
        grads = rdv.group_norm_backward(dy, x, stats, 6, w, b, activation=act)
        again = rdv.group_norm_backward(dy, x, rdv.group_norm_forward(x, 6, w, b, activation=act)[1], 6, w, b,
                                        activation=act)
        assert all(torch.equal(a, e) for a, e in zip(grads, again))
        # central differences along a direction. The step h = 2^-7 leaves h^2 of the third derivative, and the
        # float32 results' rounding over h: n^(1/2) 2^-24 / h of |dy| |y|
        for k, t in enumerate((x, w, b)):
            d = randn(g, *t.shape)
            h = 2.0 ** -7
            args = [x, w, b]
            side = []
            for s in (h, -h):
                args[k] = t + s * d
                side.append((rdv.group_norm(args[0], 6, args[1], args[2], activation=act).double() * dy).sum())
            slope, ours = (side[0] - side[1]) / (2 * h), (grads[k].double() * d).sum()
            size = (dy.double() ** 2).sum().sqrt() * (d.double() ** 2).mean().sqrt()
            assert abs(slope - ours) < 4 * h * h * size * 8 + 2.0 ** -24 / h * size * 8


def test_group_norm_refusals(rdv, cuda_device):
    x = torch.zeros(2, 5, 8, device=cuda_device)
    w = torch.zeros(8, device=cuda_device)
    for bad in (lambda: rdv.group_norm(x, 3), lambda: rdv.group_norm(x, 0), lambda: rdv.group_norm(x.double(), 2),
                lambda: rdv.group_norm(x, 2, w[:4]), lambda: rdv.group_norm(x, 2, activation="tanh"),
                lambda: rdv.group_norm(x[0, 0], 2), lambda: rdv.group_norm(x, 2, w.double()),
                lambda: rdv.group_norm_backward(x[:1], x, torch.zeros(2, 2, 2), 2),
                lambda: rdv.group_norm_backward(x, x, torch.zeros(2, 4, 2), 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(rdv.RdvbError, match="eps"):
        rdv.group_norm(x, 2, eps=-1.0)
    with pytest.raises(rdv.RdvbError, match="groups"):
        rdv.group_norm(torch.zeros(1, 2, 8192, device=cuda_device), 8192)


# ----------------------------------------------------------- cross attention


def keep_of(k, lengths, mask):
    b, lk = k.shape[:2]
    keep = torch.ones(b, lk, dtype=torch.bool, device=k.device)
    if lengths is not None:
        keep &= torch.arange(lk, device=k.device)[None] < torch.as_tensor(lengths, device=k.device)[:, None]
    return keep if mask is None else keep & mask


def attend64(q, k, v, keep, scale, dout=None):
    """Definition in 64 bits: (out, lse, and with dout dq, dk, dv), and the
    mass of each as near() takes it."""
    b, lq, h, d = q.shape
    g = h // k.shape[2]
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    qd = q.double().permute(0, 2, 1, 3)
    kd, vd = (torch.where(keep[:, :, None, None], t.double(), zero).permute(0, 2, 1, 3).repeat_interleave(g, 1)
              for t in (k, v))
    s = torch.where(keep[:, None, None], qd @ kd.transpose(-1, -2) * scale, -math.inf)
    some = keep.any(1)[:, None, None, None]
    p = torch.where(some, torch.softmax(torch.where(some, s, zero), -1), zero)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:3], -math.inf, device=q.device).double()
    res = {"out": (p @ vd, p @ vd.abs())}
    if dout is not None:
        do = dout.double().permute(0, 2, 1, 3)
        dp, delta = do @ vd.transpose(-1, -2), (do * res["out"][0]).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        mass = p * (do.abs() @ vd.abs().transpose(-1, -2) + (do.abs() * res["out"][1]).sum(-1, keepdim=True)) * abs(scale)
        shared = lambda t: t.reshape(b, -1, g, *t.shape[2:]).sum(2)  # noqa: E731
        res["dq"] = ds @ kd, mass @ kd.abs()
        res["dk"] = shared(ds.transpose(-1, -2) @ qd), shared(mass.transpose(-1, -2) @ qd.abs())
        res["dv"] = shared(p.transpose(-1, -2) @ do), shared(p.transpose(-1, -2) @ do.abs())
    return {n: tuple(t.permute(0, 2, 1, 3) for t in r) for n, r in res.items()}, lse


def check_attention(rdv, q, k, v, dout, lengths=None, mask=None, scale=None):
    keep = keep_of(k, lengths, mask)
    exact, lse64 = attend64(q, k, v, keep, q.shape[-1] ** -0.5 if scale is None else scale, dout)
    out, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths, mask=mask, scale=scale)
    near(out, exact["out"][0], q.dtype, exact["out"][1])
    assert torch.equal(torch.isinf(lse), torch.isinf(lse64))
    on = torch.isfinite(lse64)
    assert ((lse[on].double() - lse64[on]).abs() <= 64 * 2.0 ** -24 * (1 + lse64[on].abs())).all()
    only = rdv.cross_attention(q, k, v, lengths=lengths, mask=mask, scale=scale)
    near(only, exact["out"][0], q.dtype, exact["out"][1])
    grads = rdv.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths, mask=mask, scale=scale)
    for name, got in zip(("dq", "dk", "dv"), grads):
        near(got, exact[name][0], q.dtype, exact[name][1])
    assert not grads[1][~keep].any() and not grads[2][~keep].any()
    return out, grads


def inputs(seed, b, lq, lk, h, hk, d, dtype):
    g = gen(seed)
    return (randn(g, b, lq, h, d, dtype=dtype, scale=1.5), randn(g, b, lk, hk, d, dtype=dtype),
            randn(g, b, lk, hk, d, dtype=dtype), randn(g, b, lq, h, d, dtype=dtype, scale=0.1))


# b, lq, lk, heads, kv_heads, d
ATTENTION_SHAPES = [
    (1, 1, 1, 1, 1, 8), (2, 1, 700, 8, 2, 64), (1, 1, 5000, 4, 4, 128), (3, 2, 257, 6, 3, 40), (2, 5, 1, 2, 2, 64),
    (2, 63, 65, 2, 1, 16), (2, 128, 128, 2, 2, 64), (1, 129, 127, 4, 2, 128), (2, 200, 333, 8, 8, 40),
    (1, 300, 1000, 2, 2, 64), (1, 1000, 70, 4, 1, 80), (2, 100, 100, 3, 1, 33), (1, 70, 90, 2, 1, 256),
    (1, 40, 50, 2, 2, 200), (1, 7, 3000, 2, 1, 72), (2, 513, 385, 2, 2, 128), (1, 3, 2500, 16, 2, 96),
    (1, 2000, 64, 2, 2, 32), (1, 20, 130, 1, 1, 1), (4, 4, 40, 8, 1, 112)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ATTENTION_SHAPES)
def test_attention_forward_and_gradients(rdv, cuda_device, dtype, shape):
    q, k, v, dout = inputs(sum(shape), *shape, dtype)
    check_attention(rdv, q, k, v, dout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [1, 3, 150])
@pytest.mark.parametrize("d", [64, 128, 36])
def test_attention_masks_and_poison(rdv, cuda_device, dtype, lq, d):
    """Ragged lengths (0, 1, a tile's edge, past it, too long), a mask with an
    empty sample, and NaN and infinities wherever no key is allowed."""
    b, lk, h, hk = 6, 300, 4, 2
    q, k, v, dout = inputs(lq + d, b, lq, lk, h, hk, d, dtype)
    lengths = torch.tensor([0, 1, 128, 129, 300, 1000], dtype=torch.int32, device=cuda_device)
    mask = torch.rand(b, lk, generator=gen(3), device=cuda_device) < 0.7
    mask[4] = False
    mask[5, :130] = False  # whole tiles without a key
    mask[1, 0] = True
    for le, ma in ((lengths, None), (None, mask), (lengths, mask)):
        keep = keep_of(k, le, ma)
        kp, vp = k.clone(), v.clone()
        poison = torch.tensor([math.nan, math.inf, -math.inf], device=cuda_device).to(dtype)
        holes = poison[torch.arange((~keep).sum().item(), device=cuda_device) % 3][:, None, None]
        kp[~keep], vp[~keep] = holes.expand(-1, hk, d), holes.flip(0).expand(-1, hk, d)
        qp, dp = q.clone(), dout.clone()
        empty = ~keep.any(1)
        qp[empty] = math.nan  # positions of a sample without states
        out, lse = rdv.cross_attention_forward(qp, kp, vp, lengths=le, mask=ma)
        assert not out[empty].any() and (lse[empty] == -math.inf).all()
        grads = rdv.cross_attention_backward(dp, qp, kp, vp, out, lse, lengths=le, mask=ma)
        clean, clean_grads = check_attention(rdv, q, k, v, dout, le, ma)
        assert torch.equal(out, clean) and all(torch.equal(a, e) for a, e in zip(grads, clean_grads))


# b, lq, lk, heads, kv_heads, d: more items (two query tiles of a head in the forward pass, one for dQ) than processors,
# so that a block takes several; last items of one tile and of two, one to nine key tiles
WALKS = [(8, 577, 400, 8, 8, 64), (8, 576, 1000, 8, 8, 64), (8, 600, 100, 8, 4, 64), (4, 1089, 500, 16, 16, 64),
         (6, 1100, 260, 16, 4, 64), (2, 2700, 1100, 8, 8, 32), (6, 640, 300, 16, 16, 40), (8, 577, 400, 8, 8, 128),
         (6, 1300, 300, 8, 2, 128), (10, 500, 150, 8, 8, 72)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", WALKS)
def test_attention_blocks_take_several_items(rdv, cuda_device, dtype, ragged, shape):
    """What a block carries from one item to the next: barriers' phases, both
    buffers of queries, the look-ahead, and samples without states between others."""
    b, lq, lk, h = shape[:4]
    processors = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    assert -(-lq // 256) * h * b > processors
    q, k, v, dout = inputs(sum(shape) + ragged, *shape, dtype)
    lengths = mask = None
    if ragged:
        lengths = torch.tensor(([lk, 0, lk // 2, 0, 0, 1, lk - 1, 0, 129, lk])[:b], dtype=torch.int32, device=cuda_device)
        mask = torch.rand(b, lk, generator=gen(lk), device=cuda_device) < 0.8
        mask[2:3] = False  # a sample whose mask leaves nothing
    out, grads = check_attention(rdv, q, k, v, dout, lengths, mask)
    again, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths, mask=mask)
    grads_again = rdv.cross_attention_backward(dout, q, k, v, again, lse, lengths=lengths, mask=mask)
    assert torch.equal(again, out) and all(torch.equal(a, e) for a, e in zip(grads_again, grads))
    assert rdv.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("lk", [130, 1500])
def test_attention_ends_inside_a_warp(rdv, cuda_device, dtype, d, lk):
    """Rows end inside a warp's 32, positions and states alike: what lanes past the
    end skip changes nothing of the others' rows, whether parts are joined or not."""
    q, k, v, dout = inputs(d + lk, 1, 256, lk, 2, 1, d, dtype)
    dout[:, 129:] = 0
    for lq in (129, 145, 159, 255):
        out, grads = check_attention(rdv, q[:, :lq].contiguous(), k, v, dout[:, :lq].contiguous())
        if lq == 129:
            first, first_grads = out, grads
        assert torch.equal(out[:, :129], first) and torch.equal(grads[0][:, :129], first_grads[0])
    for end in (lk - 1, lk - 17):
        check_attention(rdv, q, k[:, :end], v[:, :end], dout)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_extreme_scores(rdv, cuda_device, dtype):
    """Scores far apart (one key takes all), equal scores, and scales of both
    signs and 0."""
    q, k, v, dout = inputs(11, 2, 70, 300, 2, 2, 64, dtype)
    for scale in (4.0, -1.0, 0.0, 1e-3):
        # the score's own float32 rounding grows with it: |s| 2^-24 of P, inside near()'s 64 up to |s| = 32;
        # at scale 4 scores reach 400
        exact, _ = attend64(q, k, v, keep_of(k, None, None), scale, dout)
        out, lse = rdv.cross_attention_forward(q, k, v, scale=scale)
        grads = rdv.cross_attention_backward(dout, q, k, v, out, lse, scale=scale)
        room = 1 + 8 * abs(scale)
        near(out, exact["out"][0], dtype, room * exact["out"][1])
        for name, got in zip(("dq", "dk", "dv"), grads):
            near(got, exact[name][0], dtype, room * exact[name][1])
    # the lowest finite values as keys: not a mask, just very low scores; no NaN
    low = torch.finfo(dtype).min
    k2 = k.clone()
    k2[:, 50:] = low
    out = rdv.cross_attention(q.abs() + 1, k2, v)
    few = rdv.cross_attention(q.abs() + 1, k, v, lengths=[50, 50])
    near(out, few.double(), dtype, few.double().abs() + v.double().abs().max())
    # a NaN or an infinite value that IS attended to reaches its rows
    v2 = v.clone()
    v2[0, 7, 0, 3] = math.nan
    out = rdv.cross_attention(q, k, v2)
    assert torch.isnan(out[0, :, 0, 3]).all() and torch.isfinite(out[0, :, 1]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [1, 150, 5000])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_many_small_probabilities(rdv, cuda_device, dtype, lq, d):
    """One state takes nearly all of the softmax and has no value, so that the
    result is the others', whose probabilities are equal and 2^-12 to 2^-20.5 of
    the largest: what rounding does to one it does to all. A probability in 16 bits
    keeps its digits there, u of it, and is inside near()'s two."""
    g = gen(d + lq)
    lk = 1500
    q, k, v = (torch.zeros(2, n, h, d, dtype=dtype, device=cuda_device) for n, h in ((lq, 4), (lk, 2), (lk, 2)))
    q[..., 0] = 1
    v[:] = 0.5 + randn(g, *v.shape).abs()
    v[:, 700] = 0
    for low in (12.0, 16.5, 20.5):
        k[:, 700, :, 0] = low * math.log(2)
        result, lse64 = attend64(q, k, v, keep_of(k, None, None), 1.0)
        exact, mass = result["out"]
        out, lse = rdv.cross_attention_forward(q, k, v, scale=1.0)
        near(out, exact, dtype, mass)
        assert ((lse.double() - lse64).abs() <= 64 * 2.0 ** -24 * (1 + lse64.abs())).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_small_gradients(rdv, cuda_device, dtype):
    """Gradients far below and above 1 (a scaled loss) keep their digits."""
    q, k, v, dout = inputs(13, 1, 200, 700, 2, 1, 64, dtype)
    out, lse = rdv.cross_attention_forward(q, k, v)
    for s in (2.0 ** -9, 2.0 ** 9):
        scaled = dout * s  # below 2^-14 itself rounded to float16's range: the definition takes it as it is
        exact = attend64(q, k, v, keep_of(k, None, None), 0.125, scaled)[0]
        for name, got in zip(("dq", "dk", "dv"), rdv.cross_attention_backward(scaled, q, k, v, out, lse)):
            near(got, exact[name][0], dtype, exact[name][1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lk", [1, 2, 5, 100])
@pytest.mark.parametrize("d", [40, 64, 128])
def test_attention_few_keys_gradients(rdv, cuda_device, dtype, lk, d):
    """Where few keys matter dP - delta is a small difference. Of keys within one
    tile delta is exact: dS's error is its own rounding, u |dS|, and float32's of
    what it is the difference of -- not that of the rounded output."""
    q, k, v, dout = inputs(lk + d, 2, 150, lk, 4, 2, d, dtype)
    lengths = [lk, (lk + 1) // 2]
    keep, scale = keep_of(k, lengths, None), d ** -0.5
    exact, lse64 = attend64(q, k, v, keep, scale, dout)
    out, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths)
    dq, dk, _ = rdv.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths)
    zero = torch.zeros((), dtype=torch.float64, device=cuda_device)
    qd, do = q.double().permute(0, 2, 1, 3), dout.double().permute(0, 2, 1, 3)
    kd, vd = (torch.where(keep[:, :, None, None], t.double(), zero).permute(0, 2, 1, 3).repeat_interleave(2, 1)
              for t in (k, v))
    s = torch.where(keep[:, None, None], qd @ kd.transpose(-1, -2) * scale, -math.inf)
    p = torch.softmax(s, -1)
    ds = p * (do @ vd.transpose(-1, -2) - (do * (p @ vd)).sum(-1, keepdim=True)) * scale
    own_q = ds.abs() @ kd.abs()
    own_k = (ds.abs().transpose(-1, -2) @ qd.abs()).reshape(2, 2, 2, lk, d).sum(2)
    u = U[dtype]
    for name, got, own in (("dq", dq, own_q), ("dk", dk, own_k)):
        bound = u * exact[name][0].abs() + u * own.permute(0, 2, 1, 3) + 64 * 2.0 ** -24 * exact[name][1]
        bound = bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        worst = ((got.double() - exact[name][0]).abs() / bound.clamp(min=1e-300)).max().item()
        assert worst <= 1.0, (name, worst)


def own_gradients(q, k, v, dout, keep, scale):
    """Definition in 64 bits of dS, and what dq and dk sum of its absolute values."""
    b, _, h, _ = q.shape
    g = h // k.shape[2]
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    qd, do = q.double().permute(0, 2, 1, 3), dout.double().permute(0, 2, 1, 3)
    kd, vd = (torch.where(keep[:, :, None, None], t.double(), zero).permute(0, 2, 1, 3).repeat_interleave(g, 1)
              for t in (k, v))
    s = torch.where(keep[:, None, None], qd @ kd.transpose(-1, -2) * scale, -math.inf)
    p = torch.softmax(s, -1)
    ds = (p * (do @ vd.transpose(-1, -2) - (do * (p @ vd)).sum(-1, keepdim=True)) * scale).abs()
    own_k = (ds.transpose(-1, -2) @ qd.abs()).reshape(b, -1, g, *kd.shape[2:]).sum(2)
    return (ds @ kd.abs()).permute(0, 2, 1, 3), own_k.permute(0, 2, 1, 3)


def near_own(got, exact, dtype, own):
    """got within dS's own rounding, u |dS|, and float32's of what it is the difference of."""
    u = U[dtype]
    bound = u * exact[0].abs() + u * own + 64 * 2.0 ** -24 * exact[1] + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    worst = ((got.double() - exact[0]).abs() / bound.clamp(min=1e-300)).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length", [1, 2, 5, 128])
@pytest.mark.parametrize("d", [40, 64, 128])
def test_attention_few_keys_of_long_padding(rdv, cuda_device, dtype, length, d):
    """Few states, padded to many: the long axis is split, and the gradients keep
    their digits as where it is not."""
    q, k, v, dout = inputs(length + d, 2, 150, 1000, 4, 2, d, dtype)
    lengths = [length, (length + 1) // 2]
    keep = keep_of(k, lengths, None)
    exact, _ = attend64(q, k, v, keep, d ** -0.5, dout)
    out, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths)
    dq, dk, dv = rdv.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths)
    own_q, own_k = own_gradients(q, k, v, dout, keep, d ** -0.5)
    near_own(dq, exact["dq"], dtype, own_q)
    near_own(dk, exact["dk"], dtype, own_k)
    near(dv, exact["dv"][0], dtype, exact["dv"][1])


@pytest.mark.parametrize("lq", [150, 5000])
@pytest.mark.parametrize("d,dtype", [(40, torch.float16), (40, torch.bfloat16), (64, torch.float16),
                                     (64, torch.bfloat16), (128, torch.bfloat16)])
def test_attention_one_key_of_many_matters(rdv, cuda_device, dtype, lq, d):
    """Each position all but picks one of 1000 states: dP - delta is a small
    difference there, and dK keeps its digits whether dQ's long axis is split (few
    positions) or not. Scores stay below 32, near()'s room for their rounding. Not
    float16 at 128 dimensions: there the states that are not picked have
    probabilities near 1e-9, and dS falls below the smallest step that it is held
    with, 2^-24 of 2^-E, which near_own() does not count."""
    q, k, v, dout = inputs(d, 2, lq, 1000, 4, 2, d, dtype)
    pick = torch.randint(0, 1000, (2, lq), generator=gen(d + 1), device=cuda_device)
    picked = torch.stack([k[i, pick[i]] for i in range(2)]).repeat_interleave(2, 2)
    q = (picked.float() * 2).to(dtype)
    lengths = [1000, 700]
    keep = keep_of(k, lengths, None)
    exact, _ = attend64(q, k, v, keep, d ** -0.5, dout)
    out, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths)
    _, dk, _ = rdv.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths)
    near_own(dk, exact["dk"], dtype, own_gradients(q, k, v, dout, keep, d ** -0.5)[1])


def test_attention_strides_and_streams(rdv, cuda_device):
    g = gen(21)
    kv = randn(g, 2, 150, 2, 4, 64, dtype=torch.bfloat16)
    q = randn(g, 2, 4, 90, 64, dtype=torch.bfloat16).permute(0, 2, 1, 3)  # heads outside positions
    k, v = kv[:, :, 0], kv[:, :, 1]
    dense = rdv.cross_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(rdv.cross_attention(q, k, v), dense)
    off = randn(g, 2, 150, 4, 65, dtype=torch.bfloat16)[..., 1:]  # off the 16-byte grid
    exact = attend64(q, off, v, keep_of(off, None, None), 0.125)[0]["out"]
    near(rdv.cross_attention(q, off, v), exact[0], torch.bfloat16, exact[1])
    one = k[:, :, :1].expand(-1, -1, 4, -1)  # a broadcast head
    assert torch.equal(rdv.cross_attention(q, one, v), rdv.cross_attention(q, one.contiguous(), v))
    turned = randn(g, 2, 64, 4, 150, dtype=torch.bfloat16).permute(0, 3, 2, 1)  # last dimension not dense
    assert torch.equal(rdv.cross_attention(q, turned, v), rdv.cross_attention(q, turned.contiguous(), v))
    mask = (torch.rand(2, 150, 2, generator=g, device=cuda_device) < 0.5)[..., 0]
    assert torch.equal(rdv.cross_attention(q, k, v, mask=mask), rdv.cross_attention(q, k, v, mask=mask.contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rdv.cross_attention(q, k, v)
    side.synchronize()
    assert torch.equal(other, dense)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 1248, 2372, 1, 1, 8), (2, 1100, 900, 4, 2, 64), (2, 1100, 900, 4, 1, 128)])
def test_attention_repeats_beside_other_traffic(rdv, cuda_device, dtype, shape):
    """The same bits every time while another stream keeps the memory busy, so that
    the kernels' copies arrive late and in other orders."""
    q, k, v, dout = inputs(sum(shape), *shape, dtype)
    lengths = [shape[2]] * (shape[0] - 1) + [shape[2] // 3]
    out, grads = check_attention(rdv, q, k, v, dout, torch.tensor(lengths, device=cuda_device))
    lengths = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    src = torch.zeros(2 ** 28, dtype=torch.uint8, device=cuda_device)
    dst = torch.empty_like(src)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(60):
        with torch.cuda.stream(side):
            dst.copy_(src)
        again, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths)
        grads_again = rdv.cross_attention_backward(dout, q, k, v, again, lse, lengths=lengths)
        assert torch.equal(again, out) and all(torch.equal(a, e) for a, e in zip(grads_again, grads))
    torch.cuda.current_stream().wait_stream(side)


def test_attention_lengths_of_narrow_types(rdv, cuda_device):
    q, k, v, _ = inputs(17, 3, 20, 300, 2, 1, 64, torch.bfloat16)
    values = [0, 7, 120]
    expect = rdv.cross_attention(q, k, v, lengths=torch.tensor(values, dtype=torch.int32, device=cuda_device))
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int64, torch.uint16, torch.uint32, torch.uint64):
        assert torch.equal(rdv.cross_attention(q, k, v, lengths=torch.tensor(values, dtype=dtype, device=cuda_device)), expect)


def test_attention_empty(rdv, cuda_device):
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, dout = inputs(1, b, lq, lk, 2, 1, 64, torch.float16)
        out, lse = rdv.cross_attention_forward(q, k, v)
        assert out.shape == q.shape and not out.any() and (lse == -math.inf).all()
        grads = rdv.cross_attention_backward(dout, q, k, v, out, lse)
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))


def test_attention_long_offsets(rdv, cuda_device):
    """A state sequence whose byte and element offsets pass 32 bits: only
    its far end is attended to."""
    lk, h, d = 2 ** 23 + 77, 4, 64  # 2^31 elements, 4 GiB, each of k and v
    k = torch.zeros(1, lk, h, d, dtype=torch.float16, device=cuda_device)
    v = torch.zeros(1, lk, h, d, dtype=torch.float16, device=cuda_device)
    g = gen(2)
    k[:, -500:], v[:, -500:] = randn(g, 1, 500, h, d, dtype=torch.float16), randn(g, 1, 500, h, d, dtype=torch.float16)
    mask = torch.zeros(1, lk, dtype=torch.bool, device=cuda_device)
    mask[:, -500:] = True
    for lq in (1, 40):
        q = randn(g, 1, lq, h, d, dtype=torch.float16)
        exact = attend64(q, k[:, -500:], v[:, -500:], keep_of(k[:, -500:], None, None), 0.125)[0]["out"]
        near(rdv.cross_attention(q, k, v, mask=mask), exact[0], torch.float16, exact[1])


def test_attention_last_positions(rdv, cuda_device):
    """As many states as a call takes, masked: the position after the last tile does
    not fit 31 bits. Only the end is attended to (34 GB of states, 2 GB of mask)."""
    lk, d = 2 ** 31 - 1, 8
    k = torch.zeros(1, lk, 1, d, dtype=torch.float16, device=cuda_device)
    g = gen(6)
    k[:, -500:] = randn(g, 1, 500, 1, d, dtype=torch.float16)
    mask = torch.zeros(1, lk, dtype=torch.bool, device=cuda_device)
    mask[:, -500:] = torch.rand(500, generator=g, device=cuda_device) < 0.8
    q = randn(g, 1, 40, 1, d, dtype=torch.float16)
    out = rdv.cross_attention(q, k, k, mask=mask)
    end, keep = k[:, -500:], mask[:, -500:]
    exact = attend64(q, end, end, keep, d ** -0.5)[0]["out"]
    near(out, exact[0], torch.float16, exact[1])


def test_attention_differences_and_repeats(rdv, cuda_device):
    q, k, v, dout = inputs(31, 2, 65, 130, 4, 2, 24, torch.float32)
    lengths = [130, 37]
    out, lse = rdv.cross_attention_forward(q, k, v, lengths=lengths)
    grads = rdv.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths)
    again = rdv.cross_attention_backward(dout, q, k, v, *rdv.cross_attention_forward(q, k, v, lengths=lengths),
                                         lengths=lengths)
    assert all(torch.equal(a, e) for a, e in zip(grads, again))
    g = gen(4)
    for i, t in enumerate((q, k, v)):
        d = randn(g, *t.shape)
        h = 2.0 ** -7  # as for group norm: h^2 of the third derivative, and rounding over h
        side = []
        for s in (h, -h):
            args = [q, k, v]
            args[i] = t + s * d
            side.append((rdv.cross_attention(*args, lengths=lengths).double() * dout).sum())
        slope, ours = (side[0] - side[1]) / (2 * h), (grads[i].double() * d).sum()
        size = (dout.double() ** 2).sum().sqrt()
        assert abs(slope - ours) < 32 * h * h * size + 8 * 2.0 ** -24 / h * size


def test_attention_refusals(rdv, cuda_device):
    q, k, v, dout = inputs(1, 2, 3, 5, 4, 2, 16, torch.float16)
    for bad in (lambda: rdv.cross_attention(q, k[:1], v), lambda: rdv.cross_attention(q, k, v[:, :4]),
                lambda: rdv.cross_attention(q, k.float(), v), lambda: rdv.cross_attention(q[:, :, :3], k, v),
                lambda: rdv.cross_attention(q[0], k, v), lambda: rdv.cross_attention(q.double(), k.double(), v.double()),
                lambda: rdv.cross_attention(q, k, v, lengths=[1, 2, 3]),
                lambda: rdv.cross_attention(q, k, v, lengths=[0.5, 1.0]),
                lambda: rdv.cross_attention(q, k, v, mask=torch.ones(2, 4, dtype=torch.bool)),
                lambda: rdv.cross_attention(q, k, v, mask=torch.ones(2, 5)),
                lambda: rdv.cross_attention_backward(dout[:, :2], q, k, v, q, torch.zeros(2, 4, 3)),
                lambda: rdv.cross_attention_backward(dout, q, k, v, q, torch.zeros(2, 4, 2))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(rdv.RdvbError, match="dimension"):
        rdv.cross_attention(*(t.new_zeros(*t.shape[:3], 264) for t in (q, k, v)))
    with pytest.raises(rdv.RdvbError, match="scale"):
        rdv.cross_attention(q, k, v, scale=math.inf)


# ------------------------------------------------------------------- dropout


def philox_words(seed, offset, n):
    """The Philox 4x32-10 generator in Python's whole numbers."""
    words = []
    for i in range((n + 3) // 4):
        at = (offset + i) % 2 ** 64
        c, k = [at % 2 ** 32, at >> 32, 0, 0], [seed % 2 ** 32, seed >> 32]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ c[3] ^ k[1], a % 2 ** 32]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        words += c
    return torch.tensor(words[:n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 1023, 5000])
def test_dropout_mask_and_values(rdv, cuda_device, dtype, n):
    g = gen(n)
    seed, offset, p = 2 ** 63 + 12345, 2 ** 32 - 3, 0.3
    keep = (philox_words(seed, offset, n) >= round(p * 2 ** 32)).to(cuda_device)
    x, r = randn(g, n, dtype=dtype), randn(g, n, dtype=dtype)
    zero = torch.zeros((), dtype=torch.float64, device=cuda_device)
    exact = torch.where(keep, x.double() / (1 - p), zero)
    y = rdv.dropout(x, p, seed, offset)
    assert torch.equal(y != 0, keep & (x != 0))
    near(y, exact, dtype, exact.abs(), 0)
    near(rdv.dropout(x, p, seed, offset, residual=r), exact + r.double(), dtype, exact.abs() + r.double().abs(), 0)
    assert torch.equal(rdv.dropout_backward(x, p, seed, offset), y)
    # dense but off the 16-byte grid
    room = torch.zeros(n + 1, dtype=dtype, device=cuda_device)
    room[1:] = x
    assert torch.equal(rdv.dropout(room[1:], p, seed, offset), y)
    # a dropped NaN does not pass
    assert torch.equal(torch.isnan(rdv.dropout(torch.full_like(x, math.nan), p, seed, offset)), keep)


def test_dropout_published_words():
    """Known answers of the generator (Philox 4x32-10, counter and key 0)."""
    assert philox_words(0, 0, 4).tolist() == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_dropout_rates_offsets_refusals(rdv, cuda_device):
    n = 1 << 20
    x = torch.ones(n, device=cuda_device)
    for p in (0.0, 0.1, 0.5, 0.999):
        y = rdv.dropout(x, p, 7)
        rate = (y == 0).double().mean().item()
        assert abs(rate - p) <= 6 * math.sqrt(p * (1 - p) / n)
        assert torch.equal(y[y != 0], torch.full_like(y[y != 0], 1 / (1 - p)))
    # the counter moves by four elements; other seeds are other masks
    assert torch.equal(rdv.dropout(x[:4000], 0.5, 7, 1000), rdv.dropout(x, 0.5, 7)[4000:8000])
    assert not torch.equal(rdv.dropout(x, 0.5, 7), rdv.dropout(x, 0.5, 8))
    assert rdv.dropout(x[:0], 0.5, 7).shape == (0,)
    for bad in (lambda: rdv.dropout(x, 1.0, 0), lambda: rdv.dropout(x, -0.1, 0), lambda: rdv.dropout(x, math.nan, 0),
                lambda: rdv.dropout(x, 0.1, -1), lambda: rdv.dropout(x, 0.1, 2 ** 64), lambda: rdv.dropout(x, 0.1, 0, -1),
                lambda: rdv.dropout(x, 0.1, 0, 2 ** 64 - 4), lambda: rdv.dropout(x.double(), 0.1, 0),
                lambda: rdv.dropout(x, 0.1, 0, residual=x[:5]), lambda: rdv.dropout(x, 0.1, 0, residual=x.half())):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------- autograd, tensor operations


def test_autograd_matches_explicit_gradients(rdv, cuda_device):
    g = gen(40)
    x = randn(g, 2, 12, 10, 64, dtype=torch.bfloat16).requires_grad_()
    w, b = (1 + 0.1 * randn(g, 64)).requires_grad_(), randn(g, 64).half().requires_grad_()
    dy = randn(g, 2, 12, 10, 64, dtype=torch.bfloat16)
    rdv.group_norm(x, 8, w, b, activation="silu").backward(dy)
    with torch.no_grad():
        _, stats = rdv.group_norm_forward(x, 8, w, b, activation="silu")
        grads = rdv.group_norm_backward(dy, x, stats, 8, w, b, activation="silu")
    assert all(torch.equal(t.grad, e) and t.grad.dtype == t.dtype for t, e in zip((x, w, b), grads))
    q, k, v, dout = inputs(41, 2, 30, 50, 4, 2, 64, torch.bfloat16)
    for t in (q, k, v):
        t.requires_grad_()
    out = rdv.cross_attention(q, k, v, lengths=[50, 20])
    out.backward(dout)
    with torch.no_grad():
        o, lse = rdv.cross_attention_forward(q, k, v, lengths=[50, 20])
        grads = rdv.cross_attention_backward(dout, q, k, v, o, lse, lengths=[50, 20])
    assert all(torch.equal(t.grad, e) for t, e in zip((q, k, v), grads))
    x, r = (randn(g, 1000).requires_grad_() for _ in range(2))
    dy = randn(g, 1000)
    rdv.dropout(x, 0.2, 5, 6, residual=r).backward(dy)
    assert torch.equal(x.grad, rdv.dropout_backward(dy, 0.2, 5, 6)) and torch.equal(r.grad, dy)


def test_autograd_of_wrapped_inputs(rdv, cuda_device):
    g = gen(42)
    x, dy = randn(g, 2, 30, 64), randn(g, 2, 30, 64)
    for call, shape in ((lambda t: rdv.group_norm(t, 8, activation="silu"), (2, 30, 64)),
                        (lambda t: rdv.dropout(t, 0.2, 5), (2, 30, 64)),
                        (lambda t: rdv.cross_attention(t, t, t), (2, 30, 1, 64))):
        grads = []
        for wrap in (rdv.wrap, lambda t: t):
            t = x.reshape(shape).clone().requires_grad_()
            call(wrap(t)).backward(dy.reshape(shape))
            grads.append(t.grad)
        assert torch.equal(*grads)


def test_gradients_have_their_parameters_type(rdv, cuda_device):
    g = gen(43)
    x, w = randn(g, 2, 30, 64), randn(g, 64).half()
    y, stats = rdv.group_norm_forward(x, 8, w, w)
    for param in (w, rdv.wrap(w)):
        _, dw, db = rdv.group_norm_backward(y, x, stats, 8, param, param)
        assert dw.dtype == db.dtype == torch.float16


def test_tensor_operations(rdv, cuda_device):
    g = gen(50)
    x, w, b = randn(g, 16 * 16, 32), 1 + 0.1 * randn(g, 32), randn(g, 32)
    norm = rdv.GroupNormTensorOp(x, w, b, groups=4, activation="silu")
    assert torch.equal(norm.as_type("torch"), rdv.group_norm(x[None], 4, w, b, activation="silu")[0])
    wq, bq = 0.2 * randn(g, 64, 32), torch.zeros(64, device=cuda_device)
    q = rdv.LinearTensorOp(norm, wq, bq)
    k, v = randn(g, 77, 32), randn(g, 77, 32)
    att = rdv.CrossAttentionTensorOp(q, k, v, heads=4, kv_heads=2)
    expect = rdv.cross_attention(q.as_type("torch").view(1, 256, 4, 16), k.view(1, 77, 2, 16), v.view(1, 77, 2, 16))
    assert torch.equal(att.as_type("torch"), expect.reshape(256, 64))
    before = att.as_type("torch").clone()
    x.mul_(1.7).add_(0.3 * torch.sin(x))
    att.evaluate_chain()
    assert not torch.equal(att.as_type("torch"), before)
    expect = rdv.cross_attention(q.as_type("torch").view(1, 256, 4, 16), k.view(1, 77, 2, 16), v.view(1, 77, 2, 16))
    assert torch.equal(att.as_type("torch"), expect.reshape(256, 64))
    with pytest.raises(AssertionError):
        rdv.CrossAttentionTensorOp(q, k, v, heads=3)
    with pytest.raises(AssertionError):
        rdv.GroupNormTensorOp(x, w, b, groups=5)
