"""functional.linear, functional.layer_norm and muon.newton_schulz against plain
implementations in 64 bits.

Tolerances are counted from the arithmetic, with u = 2^-24 (half a step of fp32)
and h = finfo(type).eps / 2 (half a step of the output's type):
  * a sum of K products in fp32 is off by at most (K + 2) u times the sum of the
    products' magnitudes; an affine or activation step adds a few u of its operands;
  * a 16-bit output adds h of its value; values kept in 16 bits between the two
    passes (z, dz) add h of themselves, carried on by the slopes.
Inputs that are small whole numbers make every sum exact: those tests ask for equal
values, so a wrong index, edge or stride cannot hide in a tolerance."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def half_step(t):
    return torch.finfo(t).eps / 2


def rounded(t, ref):
    """The most by which rounding to t moves ref: half a step of its value, and below the type's smallest normal number
    half of the subnormals' one step, smallest_normal * eps / 2 (fp16: 2^-14 * 2^-10 / 2 = 2^-25)."""
    return half_step(t) * ref.abs() + torch.finfo(t).smallest_normal * half_step(t)


def act64(z, act):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
            "silu": f.silu}[act](z)


def within(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    over = (got - ref).abs() - tol
    assert not torch.isnan(over).any() and float(over.max() if over.numel() else 0.0) <= 0.0, (
        f"{what}: worst |difference| {float((got - ref).abs().max()):.3e} at tolerance "
        f"{float(torch.as_tensor(tol).max()):.3e}")


def whole(shape, seed, low=-2, high=3, dtype=torch.float32):
    return torch.from_numpy(np.random.default_rng(seed).integers(low, high, shape).astype(np.float32)).to(dtype)


def normal(shape, seed, scale=1.0):
    return torch.from_numpy((scale * np.random.default_rng(seed).standard_normal(shape)).astype(np.float32))


def strided(t, lead, offset):
    """t as a view with `lead` unused columns beside it, starting `offset` elements into its storage (on the GPU)."""
    rows, cols = t.shape
    flat = torch.full((rows * (cols + lead) + offset + 8,), float("nan"), dtype=t.dtype, device="cuda")
    view = flat[offset:offset + rows * (cols + lead)].view(rows, cols + lead)[:, :cols]
    view.copy_(t)
    return view


# ----------------------------------------------------------------------------- linear
SIZES = [(1, 1, 1), (1, 64, 64), (3, 17, 5), (80, 64, 64), (16, 32, 256), (33, 130, 96), (65, 100, 515), (127, 129, 63),
         (128, 128, 128), (257, 72, 200), (300, 264, 40), (2, 1000, 1032), (17, 8, 2048), (515, 3, 7), (1030, 96, 384),
         (256, 256, 64), (255, 512, 72)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_whole_numbers_are_exact(dtype, M, N, K):
    """Forward and all gradients on whole numbers: every fp32 sum is exact, so the only rounding is the output's."""
    from sgnn_amd import functional
    x, w, b = whole((M, K), 1, dtype=dtype), whole((N, K), 2, dtype=dtype), whole((N,), 3, dtype=dtype)
    r, dy = whole((M, N), 4, dtype=dtype), whole((M, N), 5, dtype=dtype)
    for act, res in (("none", None), ("relu", None), ("relu", r), ("none", r)):
        z = x.double() @ w.double().T + b.double()
        y = (act64(z, act) + (0.0 if res is None else res.double())).to(dtype)
        dz = dy.double() * (z > 0) if act == "relu" else dy.double()
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b) + ((r,) if res is not None else ())]
        got = functional.linear(*leaves[:3], activation=act, residual=leaves[3] if res is not None else None)
        grads = torch.autograd.grad(got, leaves, dy.cuda())
        what = f"{act} residual={res is not None}"
        assert torch.equal(got.detach().cpu(), y), what
        for name, g, ref in zip(("dx", "dw", "db", "dres"), grads,
                                (dz @ w.double(), dz.T @ x.double(), dz.sum(0), dy.double())):
            assert torch.equal(g.cpu(), ref.to(dtype)), f"{what} {name}"
        with torch.no_grad():
            again = functional.linear(*leaves[:3], activation=act, residual=leaves[3] if res is not None else None)
        assert torch.equal(again, got.detach()), what


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lead,offset", [(0, 1), (1, 0), (3, 5), (8, 0), (8, 8)])
def test_linear_strides_and_alignment(dtype, lead, offset):
    """Operands with unused columns, at storage offsets that no vector is aligned to: what lies between the rows is
    never read into a result (it is NaN here)."""
    from sgnn_amd import functional
    M, N, K = 70, 75, 88
    x, w, r, dy = (whole(s, i, dtype=dtype) for i, s in enumerate([(M, K), (N, K), (M, N), (M, N)]))
    xs, wsd, rs, dys = (strided(t, lead, offset) for t in (x, w, r, dy))
    leaves = [t.requires_grad_(True) for t in (xs, wsd, rs)]
    got = functional.linear(leaves[0], leaves[1], None, "relu", leaves[2])
    dx, dw, dres = torch.autograd.grad(got, leaves, dys)
    z = x.double() @ w.double().T
    dz = dy.double() * (z > 0)
    assert torch.equal(got.detach().cpu(), (z.relu() + r.double()).to(dtype))
    assert torch.equal(dx.cpu(), (dz @ w.double()).to(dtype)) and torch.equal(dw.cpu(), (dz.T @ x.double()).to(dtype))
    assert torch.equal(dres.cpu(), dy)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(70, 80, 72), (200, 136, 200), (24, 40, 4168), (1000, 136, 72), (4000, 3200, 72)])
def test_linear_has_the_same_bits_at_any_alignment(dtype, M, N, K):
    """Dense operands, and views that start one element further on or have unused columns: the summation order depends on
    the sizes alone (sizes whose last block of k is a part of one, in every product)."""
    from sgnn_amd import functional
    x, w, dy = normal((M, K), 1).to(dtype), normal((N, K), 2, K ** -0.5).to(dtype), normal((M, N), 3).to(dtype)
    runs = []
    for lead, offset in ((0, 0), (0, 1), (1, 0), (8, 8)):
        xs, wsd, dys = (strided(t, lead, offset) for t in (x, w, dy))
        for act in ("none", "silu"):
            leaves = [xs.requires_grad_(True), wsd.requires_grad_(True)]
            y = functional.linear(*leaves, None, act)
            runs.append((act, lead, offset, [y.detach(), *torch.autograd.grad(y, leaves, dys)]))
    for act, lead, offset, got in runs[2:]:
        want = next(r for r in runs if r[0] == act)[3]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (act, lead, offset)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_has_the_same_bits_at_any_leading_dimension(dtype):
    """Rows far apart (2^22 elements and more) are loaded by another path than near ones, in the same order of k."""
    from sgnn_amd import functional
    M, N, K, ld = 40, 48, 72, (1 << 22) + 64
    x, w, dy = normal((M, K), 1).to(dtype).cuda(), normal((N, K), 2).to(dtype).cuda(), normal((M, N), 3).to(dtype).cuda()
    far = torch.zeros(M, ld, dtype=dtype, device="cuda")
    far[:, :K] = x
    outs = []
    for a in (x, far[:, :K]):
        leaves = [a.requires_grad_(True), w.requires_grad_(True)]
        y = functional.linear(*leaves)
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(37, 50, 70), (130, 140, 260), (1, 96, 600)])
def test_linear_against_64_bits(dtype, act, M, N, K):
    from sgnn_amd import functional
    h = half_step(dtype)
    h16 = h if dtype != torch.float32 else 0.0   # of values kept in the type between the passes
    x, w, b, r, dy = (t.to(dtype) for t in (normal((M, K), 1), normal((N, K), 2, K ** -0.5), normal((N,), 3),
                                            normal((M, N), 4), normal((M, N), 5)))
    z = x.double() @ w.double().T + b.double()
    if act == "relu":   # keep every z far enough from the slope's jump
        x = x.clone()
        b = (b.double() + 40.0 * (torch.arange(N) % 2 * 2 - 1)).to(dtype)
        z = x.double() @ w.double().T + b.double()
        assert float(z.abs().min()) > 1.0
    d = [t.double().requires_grad_(True) for t in (x, w, b, r)]
    ref = act64(d[0] @ d[1].T + d[2], act) + d[3]
    ref_grads = torch.autograd.grad(ref, d, dy.double())
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, r)]
    got = functional.linear(*leaves[:3], activation=act, residual=leaves[3])
    grads = torch.autograd.grad(got, leaves, dy.cuda())
    # z, then the activation (slope at most 1.13; its functions good to (|z| + 8) 2 u of |z|), then the residual
    mags = x.double().abs() @ w.double().abs().T + b.double().abs()
    ez = (K + 4) * U * mags
    ey = 1.13 * ez + (z.abs() + 8) * 2 * U * z.abs() + 2 * U * (z.abs() + r.double().abs())
    within(got, ref.detach(), ey * (1 + h) + rounded(dtype, ref.detach()), f"y {act}")
    # dz: slopes change by at most 0.8 per unit of z (nothing for none and relu, away from 0)
    bend = 0.0 if act in ("none", "relu") else 0.8
    slope = torch.autograd.grad(act64(zz := z.clone().requires_grad_(True), act).sum(), zz)[0]
    dz = dy.double() * slope
    edz = dy.double().abs() * (bend * (ez + h16 * z.abs()) + (z.abs() + 8) * 8 * U) + (h16 > 0) * rounded(dtype, dz) * (act != "none")
    ad, aw, ax = dz.abs(), w.double().abs(), x.double().abs()
    tols = ((N + 4) * U * (ad @ aw) + edz @ aw, (M + 4) * U * (ad.T @ ax) + edz.T @ ax,
            (M + 4) * U * ad.sum(0) + edz.sum(0), 0.0)
    for name, g, rg, tol in zip(("dx", "dw", "db", "dres"), grads, ref_grads, tols):
        within(g, rg, tol * (1 + h) + rounded(dtype, rg) * (name != "dres"), f"{name} {act}")


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,N,K", [(37, 50, 70), (24, 72, 64), (130, 136, 264), (200, 328, 2056), (260, 515, 771), (3600, 72, 3600),
                                   (72, 3600, 3600), (20011, 40, 24), (5000, 136, 200)])
def test_linear_gradients_are_rounded_once(dtype, act, M, N, K):
    """dz keeps h^2 of itself (two halves of h each) and 2^-36 where it is small, so a 16-bit gradient is off by its own
    rounding and what fp32 sums lose.  Slopes: (|z| + 8) 8 u as in the test above, 7.5e-8 for gelu's distribution function,
    and 0.8 times the error of z."""
    from sgnn_amd import functional
    h = half_step(dtype)
    x, w, b, dy = (t.to(dtype).cuda() for t in (normal((M, K), 1), normal((N, K), 2, K ** -0.5), normal((N,), 3),
                                                normal((M, N), 4)))
    wide = lambda t: t.detach().double()
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(functional.linear(*leaves, act), leaves, dy)
    z = (wide(x) @ wide(w).T + wide(b)).requires_grad_(True)
    slope, = torch.autograd.grad(act64(z, act).sum(), z)
    z, dz = z.detach(), dy.double() * slope
    ez = (K + 4) * U * (wide(x).abs() @ wide(w).abs().T + wide(b).abs())
    edz = dy.double().abs() * (0.8 * ez + (z.abs() + 8) * 8 * U + 7.5e-8) + h * h * dz.abs() + 2.0 ** -36
    ad, aw, ax = dz.abs(), wide(w).abs(), wide(x).abs()
    for name, got, ref, tol in (("dx", dx, dz @ wide(w), (N + 4) * 2 * U * (ad @ aw) + edz @ aw),
                                ("dw", dw, dz.T.contiguous() @ wide(x), (M + 4) * 2 * U * (ad.T.contiguous() @ ax) + edz.T.contiguous() @ ax),
                                ("db", db, dz.sum(0), (M + 4) * U * ad.sum(0) + edz.sum(0))):
        within(got, ref.cpu(), (tol * (1 + h) + rounded(dtype, ref)).cpu(), f"{name} {act}")


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
def test_linear_gradients_past_the_largest_value(dtype):
    """dz = dy act'(z), with dy the type's largest value and a slope of 1.1, does not fit the type; dx = dz w does."""
    from sgnn_amd import functional
    x = torch.full((20, 3), 51.0, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.full((1, 3), 2.0 ** -6, dtype=dtype, device="cuda")
    dy = torch.full((20, 1), torch.finfo(dtype).max, dtype=dtype, device="cuda")
    z = (x.detach().double() @ w.double().T).requires_grad_(True)
    slope, = torch.autograd.grad(torch.nn.functional.silu(z).sum(), z)
    assert float(slope.min()) > 1.08
    dx, = torch.autograd.grad(functional.linear(x, w, None, "silu"), x, dy)
    ref = dy.double() * slope @ w.double()
    # the slope to 100 u (of the same size), on top of the rounding
    within(dx, ref.cpu(), ((half_step(dtype) + 100 * U) * ref).cpu(), "dx")


@pytest.mark.parametrize("act", ["relu", "silu"])
def test_linear_backward_of_very_many_columns(act):
    """Nine million output features (and terms of dx).  relu: whole numbers, exact; silu: dz to 2^-16 of itself, sums of 9e6 products by 32 and by splits."""
    from sgnn_amd import functional
    M, N, t = 2, 9_000_000, torch.bfloat16
    x, w, dy = (whole(s, i, -1, 2, dtype=t).cuda() for i, s in enumerate([(M, 1), (N, 1), (M, N)]))
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    dx, dw = torch.autograd.grad(functional.linear(*leaves, None, act), leaves, dy)
    z = (x.detach().double() @ w.detach().double().T).requires_grad_(True)
    slope, = torch.autograd.grad(act64(z, act).sum(), z)
    dz = dy.double() * slope
    for g, ref, mags in ((dx, dz @ w.detach().double(), dz.abs() @ w.detach().double().abs()),
                         (dw, dz.T.contiguous() @ x.detach().double(), dz.abs().T.contiguous() @ x.detach().double().abs())):
        if act == "relu":
            assert torch.equal(g, ref.to(t))
        else:
            within(g, ref.cpu(), (rounded(t, ref) * 1.01 + (2.0 ** -16 + (9e6 / 256 / 32 + 60) * U) * mags).cpu(), act)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(70, 75, 88), (300, 264, 40), (1030, 96, 384)])
def test_linear_by_c_with_slopes_of_0_and_1(dtype, M, N, K):
    """relu's slopes with and without SGNN_SLOPES_01: exact on whole numbers, the tiniest values among them."""
    dy, x, w = (whole(s, i, dtype=dtype).cuda() for i, s in enumerate([(M, N), (M, K), (N, K)]))
    slope = whole((M, N), 9, 0, 2).cuda()
    dy[3], dy[:, 5], dy[3, 5], slope[3, 5] = 0, 0, 3 * 2.0 ** -24, 1   # alone in its sums; its half is no fp16 value
    dz = dy.double() * slope.double()
    want = [t.to(dtype) for t in (dz @ w.double(), dz.T.contiguous() @ x.double(), dz.sum(0))]
    for flags in (0, 0x100):
        for got, ref in zip(_linear_bwd_by_c(dy, slope, x, w, flags), want):
            assert torch.equal(got, ref), flags


def _linear_bwd_by_c(dy, slope, x, w, flags=0):
    from sgnn_amd import _hip
    L = _hip.lib()
    (M, N), K, dt = dy.shape, x.shape[1], _hip.DTYPES[x.dtype] | flags
    nws = L.sgnn_linear_bwd_workspace_bytes(dt, M, N, K, int(slope is not None))
    ws = torch.empty(nws, dtype=torch.uint8, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(N, dtype=x.dtype, device="cuda")
    _hip.check(L.sgnn_linear_bwd(dt, M, N, K, dy.data_ptr(), N, slope.data_ptr() if slope is not None else None,
                                 x.data_ptr(), K, w.data_ptr(), K, dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                 ws.data_ptr(), nws, torch.cuda.current_stream().cuda_stream), "sgnn_linear_bwd")
    return dx, dw, db


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(4, 20, 24), (70, 75, 88), (300, 264, 40), (70, 33, 4100), (5, 6, 0)])
def test_linear_by_c_writes_every_slope(dtype, M, N, K):
    """A slope buffer is written whatever the activation: ones without one, and relu's 0 and 1; the gradients that read
    it are those without a buffer."""
    from sgnn_amd import _hip
    L, dt = _hip.lib(), _hip.DTYPES[dtype]
    x, w, dy = (whole(s, i, dtype=dtype).cuda() for i, s in enumerate([(M, K), (N, K), (M, N)]))
    nws = L.sgnn_linear_workspace_bytes(dt, M, N, K)
    ws = torch.empty(max(nws, 1), dtype=torch.uint8, device="cuda")
    for act, want in (("none", torch.ones(M, N)), ("relu", (x.double() @ w.double().T > 0).float().cpu())):
        y, slope = torch.empty(M, N, dtype=dtype, device="cuda"), torch.full((M, N), 7.0, device="cuda")
        _hip.check(L.sgnn_linear(dt, M, N, K, x.data_ptr(), K, w.data_ptr(), K, None, _hip.ACTIVATIONS[act], None, 0,
                                 slope.data_ptr(), y.data_ptr(), N, ws.data_ptr(), nws,
                                 torch.cuda.current_stream().cuda_stream), "sgnn_linear")
        assert torch.equal(slope.cpu(), want), act
        if act == "none" and K:
            for a, b in zip(_linear_bwd_by_c(dy, slope, x, w), _linear_bwd_by_c(dy, None, x, w)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("K", [48, 50])
def test_linear_gradients_non_finite_values_propagate(dtype, K):
    """An infinity or NaN of w, x or dy reaches the gradients that read it as 64-bit arithmetic has it (slopes of 0.3: dz
    is no value of a 16-bit type)."""
    M, N = 40, 72
    dy, x, w = (whole(s, i, 1, 4, dtype=dtype) for i, s in enumerate([(M, N), (M, K), (N, K)]))
    w[11, 2], w[30, 7], x[7, 9], x[3, 5], dy[20, 40] = float("inf"), float("nan"), float("-inf"), float("nan"), float("inf")
    slope = torch.full((M, N), 0.3)
    dz = dy.double() * slope.double()
    got = _linear_bwd_by_c(*(t.cuda() for t in (dy, slope, x, w)))
    for name, g, ref in zip(("dx", "dw", "db"), got, (dz @ w.double(), dz.T @ x.double(), dz.sum(0))):
        g = g.double().cpu()
        assert torch.equal(g.isnan(), ref.isnan()) and torch.equal(g.isinf(), ref.isinf()), name
        assert torch.equal(g[g.isinf()] > 0, ref[ref.isinf()] > 0), name
        fine = ref.isfinite()
        # sums of at most 72 positive terms; dz to 2^-16
        within(g[fine], ref[fine], (half_step(dtype) + 2.0 ** -16 + 80 * U) * ref[fine], name)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act,low,high", [("silu", -16.0, -8.0), ("gelu", -6.0, -4.0), ("gelu_tanh", -6.0, -4.0),
                                          ("silu", 8.0, 16.0), ("gelu", 4.0, 6.0)])
def test_linear_gradients_in_the_tails(dtype, act, low, high):
    """z = x exactly (one feature of weight 1), far out where a slope is a small fraction of 1: dx = dy act'(z) to half a
    step of its own size.  The functions: exp is good to (its argument + 8) 2 u, the normal distribution function to
    7.5e-8 (16-bit types) or 4 u, and the sums of a slope's terms add 4 u of each."""
    from sgnn_amd import functional
    x = torch.linspace(low, high, 301).to(dtype)[:, None]
    dy = (64.0 * normal((301, 1), 1)).to(dtype)
    z = x.double().requires_grad_(True)
    slope, = torch.autograd.grad(act64(z, act).sum(), z)
    z = z.detach()
    if act == "silu":
        fn = torch.sigmoid(z) * (1 + z.abs()) * (z.abs() + 8) * 6 * U
    elif act == "gelu":
        pdf = torch.exp(-0.5 * z * z) / (2 * np.pi) ** 0.5
        fn = (7.5e-8 if dtype != torch.float32 else 4 * U) + z.abs() * pdf * (0.5 * z * z + 8) * 6 * U + 4 * U * (z > 0)
    else:
        u = 2 * (2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)
        fn = torch.sigmoid(u) * (1 + z.abs() * 1.6 * (1 + 0.134145 * z * z)) * (u.abs() + 8) * 6 * U
    xg, w = x.cuda().requires_grad_(True), torch.ones(1, 1, dtype=dtype, device="cuda")
    dx, = torch.autograd.grad(functional.linear(xg, w, None, act), xg, dy.cuda())
    ref = dy.double() * slope
    within(dx, ref, dy.double().abs() * fn * (1 + half_step(dtype)) + rounded(dtype, ref) * (1 + 2.0 ** -10), act)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_long_reduction(dtype):
    """The weight's gradient of many rows, and its bias', are whole-number exact (each partial sum < 2^24)."""
    from sgnn_amd import functional
    M, N, K = 20011, 40, 24
    x, w, dy = whole((M, K), 1, dtype=dtype), whole((N, K), 2, dtype=dtype), whole((M, N), 3, dtype=dtype)
    b = torch.zeros(N, dtype=dtype)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(functional.linear(*leaves), leaves, dy.cuda())
    assert torch.equal(dw.cpu(), (dy.double().T @ x.double()).to(dtype))
    assert torch.equal(db.cpu(), dy.double().sum(0).to(dtype))
    assert torch.equal(dx.cpu(), (dy.double() @ w.double()).to(dtype))


@pytest.mark.parametrize("M,N,K,what", [(4096, 2048, 4096, "y"), (1000003, 64, 64, "dw"), (2048, 2048, 2048, "dx"), (20, 300, 4096, "y")])
def test_linear_fp32_sums_of_positive_values(M, N, K, what):
    """Products that all add up, as behind a ReLU: a sum by 32 k at a time is off by at most u of each partial sum, half
    of the whole on the average, and 36 u within its blocks (32 products, six parts); at most 256 splits are added by
    eights of 32."""
    from sgnn_amd import functional
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, w, dy = (torch.rand(*s, generator=gen, device="cuda").requires_grad_(True) for s in ((M, K), (N, K), (M, N)))
    y = functional.linear(x, w)
    wide = lambda t: t.detach().double()
    if what == "y":
        got, ref, k = y.detach(), wide(x) @ wide(w).T.contiguous(), K
    else:
        got, = torch.autograd.grad(y, x if what == "dx" else w, dy.detach())
        ref, k = (wide(dy) @ wide(w), N) if what == "dx" else (wide(dy).T.contiguous() @ wide(x), M)
    adds = min(k / 32 / 2, k / 256 / 32 / 2 + 20) if k > 1 << 18 else k / 32 / 2
    worst = float(((got.double() - ref).abs() / ref).max())
    print(f"worst {worst:.2e} at {(adds + 36) * U:.2e}")
    assert worst <= (adds + 36) * U


def test_linear_gradient_against_differences():
    """fp32 gradients against central differences of the operator's own sum, in a direction of each input."""
    from sgnn_amd import functional
    t = [normal(s, i, 0.5).cuda() for i, s in enumerate([(9, 20), (13, 20), (13,), (9, 13)])]
    dirs = [normal(tuple(v.shape), 50 + i).cuda() for i, v in enumerate(t)]
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [v.clone().requires_grad_(True) for v in t]
        grads = torch.autograd.grad(functional.linear(*leaves[:3], act, leaves[3]).double().sum(), leaves)
        for i in range(4):
            def value(step):
                args = [v + step * dirs[i] if j == i else v for j, v in enumerate(t)]
                return float(functional.linear(*args[:3], act, args[3]).double().sum())
            e = 2.0 ** -6
            diff = (value(e) - value(-e)) / (2 * e)
            # 9 * 13 outputs of magnitude < 16, each off by < 64 u of it; a third derivative of magnitude < 2 along
            # the direction, whose size per output is < 12: e^2 / 6 * 2 * 12^3 per output at the very worst
            tol = 117 * 16 * 64 * U / e + 117 * e * e / 6 * 2 * 12 ** 3 * 0.01
            assert abs(diff - float((grads[i].double() * dirs[i].double()).sum())) <= tol, (act, i)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(3841, 3080, 40), (3841, 3081, 41), (8200, 1000, 1030), (8200, 1000, 1032),
                                   (30, 700, 300), (32, 4096, 1100), (25, 33, 4100)])
def test_linear_of_many_tiles_is_exact(dtype, M, N, K):
    """The largest tiles with ragged edges, and some rows against wide weights (|sums| <= 4 * 8200 < 2^24)."""
    from sgnn_amd import functional
    x, w, dy = (whole(s, i, dtype=dtype).cuda() for i, s in enumerate([(M, K), (N, K), (M, N)]))
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    got = functional.linear(*leaves, activation="relu")
    dx, dw = torch.autograd.grad(got, leaves, dy)
    z = x.detach().double() @ w.detach().double().T
    dz = dy.double() * (z > 0)
    assert torch.equal(got.detach(), z.relu().to(dtype))
    assert torch.equal(dx, (dz @ w.detach().double()).to(dtype))
    assert torch.equal(dw, (dz.T.contiguous() @ x.detach().double()).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_linear_offsets_past_32_bits(dtype):
    """Rows 20M elements apart, and 2^31 elements of x: whole numbers, so the far rows are exact."""
    from sgnn_amd import functional
    rows, K, N, ld = 130, 72, 40, 20_000_000
    x, w, dy = whole((rows, K), 1, dtype=dtype), whole((N, K), 2, dtype=dtype), whole((rows, N), 3, dtype=dtype)
    far = torch.empty(rows * ld, dtype=dtype, device="cuda").view(rows, ld)
    xs, dys = far[:, :K], far[:, 100:100 + N]
    xs.copy_(x), dys.copy_(dy)
    leaves = [xs.detach().requires_grad_(True), w.cuda().requires_grad_(True)]
    got = functional.linear(*leaves, residual=dys)
    dx, dw = torch.autograd.grad(got, leaves, dys)
    assert torch.equal(got.detach().cpu(), (x.double() @ w.double().T + dy.double()).to(dtype))
    assert torch.equal(dx.cpu(), (dy.double() @ w.double()).to(dtype))
    assert torch.equal(dw.cpu(), (dy.double().T @ x.double()).to(dtype))
    y = functional.layer_norm(xs)
    assert torch.equal(y, functional.layer_norm(xs.contiguous()))
    del far, xs, dys, leaves, got, dx, dw
    M = 2 ** 31 // K + 1000
    tall = torch.zeros(M, K, dtype=dtype, device="cuda")
    tall[-rows:] = x.cuda()
    assert torch.equal(functional.linear(tall, w.cuda())[-rows:].cpu(), (x.double() @ w.double().T).to(dtype))
    ones = torch.ones(K, dtype=dtype, device="cuda").requires_grad_(True)
    leaf = tall.requires_grad_(True)
    out = functional.layer_norm(leaf, ones)
    assert torch.equal(out.detach()[-rows:], functional.layer_norm(x.cuda(), ones.detach()))
    dx, = torch.autograd.grad(out, leaf, tall.detach())
    few = x.cuda().requires_grad_(True)
    want, = torch.autograd.grad(functional.layer_norm(few, ones), few, x.cuda())
    assert torch.equal(dx[-rows:], want) and not dx[:-rows].any()


def test_linear_edges_of_sizes():
    from sgnn_amd import functional
    for dtype in TYPES:
        w, b = whole((6, 4), 1, dtype=dtype).cuda().requires_grad_(True), whole((6,), 2, dtype=dtype).cuda().requires_grad_(True)
        x = torch.empty(0, 4, dtype=dtype, device="cuda", requires_grad=True)
        y = functional.linear(x, w, b, "gelu")
        assert y.shape == (0, 6)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 6, dtype=dtype, device="cuda"))
        assert dx.shape == (0, 4) and not dw.any() and not db.any()
        assert functional.linear(x.detach(), w[:0]).shape == (0, 0)
        # no input features: the bias alone
        x0, w0 = torch.empty(5, 0, dtype=dtype, device="cuda"), torch.empty(6, 0, dtype=dtype, device="cuda")
        assert torch.equal(functional.linear(x0, w0, b.detach(), "relu"), b.detach().relu().expand(5, 6))
        # leading dimensions, one vector, an expanded row, a transposed matrix
        x3 = whole((2, 3, 4), 5, dtype=dtype).cuda()
        ref = (x3.double() @ w.detach().double().T).to(dtype)
        assert torch.equal(functional.linear(x3, w.detach()), ref)
        assert torch.equal(functional.linear(x3[0, 0], w.detach()), ref[0, 0])
        row = x3[0, :1].expand(7, 4)
        assert torch.equal(functional.linear(row, w.detach()), ref[0, :1].expand(7, 6))
        xt = x3[0].t().contiguous().t()
        assert torch.equal(functional.linear(xt, w.detach()), ref[0])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M", [0, 5])
def test_linear_without_outputs_has_gradients(dtype, M):
    """No output features: y is [M, 0], the input's gradient a sum of nothing, the weight's and the bias' empty."""
    from sgnn_amd import functional
    x = torch.ones(M, 4, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.ones(0, 4, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.ones(0, dtype=dtype, device="cuda", requires_grad=True)
    for act in ("none", "silu"):
        y = functional.linear(x, w, b, act)
        assert y.shape == (M, 0)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(M, 0, dtype=dtype, device="cuda"))
        assert torch.equal(dx, torch.zeros_like(x)) and dw.shape == (0, 4) and db.shape == (0,)


def test_linear_non_finite_values_propagate():
    """A NaN or infinity reaches exactly the outputs that read it, as fp32 arithmetic has it; ReLU keeps a NaN."""
    from sgnn_amd import functional
    for dtype in TYPES:
        x, w = whole((40, 48), 1, 1, 4, dtype=dtype), whole((72, 48), 2, 1, 4, dtype=dtype)
        x[3, 5], x[7, 9], x[8, 47], w[11, 2] = float("nan"), float("inf"), float("-inf"), float("inf")
        ref = x.double() @ w.double().T
        for act in ("none", "relu"):
            got = functional.linear(x.cuda(), w.cuda(), activation=act).cpu().double()
            want = ref if act == "none" else torch.where(ref < 0, torch.zeros_like(ref), ref)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1.5, 1e9, -1e9),
                                                                          want.to(dtype).double().nan_to_num(1.5, 1e9, -1e9))


def test_linear_of_nan_costs_no_multiple_of_the_product():
    """A diverged fp32 step (every output NaN) is formed once more by matrix instructions: far below the more than
    hundred times that one lane per output took.  Forward, dx and dw."""
    from sgnn_amd import functional
    n = 2048

    def step(x, w, dy):
        leaves = [x.requires_grad_(True), w.requires_grad_(True)]
        y = functional.linear(*leaves)
        return y, *torch.autograd.grad(y, leaves, dy)

    def best(args):
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            step(*args)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    args = [normal((n, n), i).cuda() for i in range(3)]
    finite = best(args)
    args[1].detach()[5, 7] = float("nan")
    one = best(args)
    bad = [torch.full_like(t, float("nan")) for t in args]
    assert all(t.isnan().all() for t in step(*bad))
    every = best(bad)
    print(f"finite {finite:.3f} ms, one NaN {one:.3f} ms, all NaN {every:.3f} ms")
    assert one <= 4 * finite + 1.0 and every <= 40 * finite


def test_linear_refuses():
    from sgnn_amd import functional
    x, w = torch.zeros(3, 4, device="cuda"), torch.zeros(5, 4, device="cuda")
    bad = [lambda: functional.linear(x.double(), w.double()), lambda: functional.linear(x, w.bfloat16()),
           lambda: functional.linear(x, w.t()), lambda: functional.linear(x, w, torch.zeros(4, device="cuda")),
           lambda: functional.linear(x, w, torch.zeros(5)), lambda: functional.linear(x, w, activation="tanh"),
           lambda: functional.linear(x, w, residual=torch.zeros(3, 4, device="cuda")),
           lambda: functional.linear(x, w, residual=torch.zeros(5, device="cuda")),
           lambda: functional.linear(x, w[0])]
    for call in bad:
        with pytest.raises(ValueError):
            call()


# ----------------------------------------------------------------------------- layer norm
LN_SIZES = [(1, 1), (1, 64), (2, 3), (80, 64), (5, 128), (513, 96), (33, 100), (7, 771), (300, 256), (64, 1000),
            (9, 4096), (3, 5003), (2, 8192), (4, 9000), (1000, 16), (129, 24), (2, 20000)]


def _ln64(x, w, b, r, eps):
    y = torch.nn.functional.layer_norm(x, (x.shape[-1],), w, b, eps)
    return y if r is None else y + r


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n,width", LN_SIZES)
@pytest.mark.parametrize("w32", [False, True])
def test_layer_norm_against_64_bits(dtype, n, width, w32):
    from sgnn_amd import functional
    wtype = torch.float32 if w32 else dtype
    h, eps = half_step(dtype), 1e-5
    x = (normal((n, width), 1, 2.0) + 1.5).to(dtype)
    w, b = (1.0 + normal((width,), 2, 0.2)).to(wtype), normal((width,), 3, 0.3).to(wtype)
    r, dy = normal((n, width), 4).to(dtype), normal((n, width), 5).to(dtype)
    for res in (None, r):
        given = [x, w, b] + ([r] if res is not None else [])
        d = [t.double().requires_grad_(True) for t in given]
        ref = _ln64(*d[:3], d[3] if res is not None else None, eps)
        ref_grads = torch.autograd.grad(ref, d, dy.double())
        leaves = [t.cuda().requires_grad_(True) for t in given]
        got = functional.layer_norm(*leaves[:3], residual=leaves[3] if res is not None else None, eps=eps)
        grads = torch.autograd.grad(got, leaves, dy.cuda())
        x64, w64, up = x.double(), w.double(), dy.double()
        mean = x64.mean(1, keepdim=True)
        rstd = 1.0 / (x64.var(1, unbiased=False, keepdim=True) + eps).sqrt()
        hat = (x64 - mean) * rstd
        # a row sum: at most width / 8 + 16 additions deep
        c = (width / 8 + 16) * U
        emean = c * x64.abs().mean(1, keepdim=True)
        ehat = rstd * (emean + 2 * U * (x64.abs() + mean.abs())) + hat.abs() * (c + 8 * U) + hat.abs() * rstd ** 2 * emean ** 2
        ey = w64.abs() * ehat + 4 * U * ((hat * w64).abs() + b.double().abs() + (res.double().abs() if res is not None else 0))
        within(got, ref.detach(), ey * (1 + h) + rounded(dtype, ref.detach()), "y")
        g = up * w64
        gm, ghm = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
        agm, aghm = g.abs().mean(1, keepdim=True), (g * hat).abs().mean(1, keepdim=True)
        egm = c * agm
        eghm = c * aghm + (g.abs() * ehat).mean(1, keepdim=True)
        inner = g - gm - hat * ghm
        edx = rstd * (egm + hat.abs() * eghm + ehat * ghm.abs() + 6 * U * (g.abs() + gm.abs() + (hat * ghm).abs())) \
            + (c + 16 * U) * rstd * inner.abs() + rstd ** 3 * emean ** 2 * inner.abs()
        edw = (n + 4) * U * (up * hat).abs().sum(0) + (up.abs() * ehat).sum(0)
        edb = (n + 4) * U * up.abs().sum(0)
        for name, gr, rg, tol in zip(("dx", "dw", "db", "dres"), grads, ref_grads, (edx, edw, edb, 0.0)):
            kind = wtype if name in ("dw", "db") else dtype
            assert gr.dtype == kind
            within(gr, rg, tol * (1 + half_step(kind)) + rounded(kind, rg) * (name != "dres"), name)
        with torch.no_grad():
            again = functional.layer_norm(*leaves[:3], residual=leaves[3] if res is not None else None, eps=eps)
        assert torch.equal(again, got.detach())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("lead,offset", [(0, 1), (1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("width", [72, 88, 203, 1024])
def test_layer_norm_strides_and_alignment(dtype, lead, offset, width):
    """The same bits from strided, unaligned rows as from dense ones."""
    from sgnn_amd import functional
    x, r, dy = (normal((50, width), i).to(dtype) for i in range(3))
    w, b = normal((width,), 4).to(dtype).cuda().requires_grad_(True), normal((width,), 5).to(dtype).cuda().requires_grad_(True)
    outs = []
    for make in (lambda t: t.cuda(), lambda t: strided(t, lead, offset)):
        xs, rs, dys = make(x).requires_grad_(True), make(r).requires_grad_(True), make(dy)
        y = functional.layer_norm(xs, w, b, residual=rs)
        outs.append([y.detach(), *torch.autograd.grad(y, (xs, w, b, rs), dys)])
    h = half_step(dtype)
    for a, c in zip(*outs):
        # the lanes' share of a row may differ with the alignment: at most a last step of the output's type apart
        within(a, c.double().cpu(), (2 * h + 64 * U) * (c.double().cpu().abs() + (0 if h > U else c.double().cpu().abs().max())), "strided")


def test_layer_norm_without_weights_and_edges():
    from sgnn_amd import functional
    x = normal((6, 40), 1).cuda()
    ref = _ln64(x.double(), None, None, None, 1e-5).cpu()
    within(functional.layer_norm(x), ref, 64 * U * (1 + ref.abs()), "no weights")
    w = normal((40,), 2).cuda()
    within(functional.layer_norm(x, w), ref * w.double().cpu(), 64 * U * (1 + ref.abs()) * w.double().cpu().abs(), "no bias")
    within(functional.layer_norm(x, None, w), ref + w.double().cpu(), 64 * U * (1 + ref.abs() + w.double().cpu().abs()), "no weight")
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, db = torch.autograd.grad(functional.layer_norm(xg, None, wg).sum(), (xg, wg))
    within(db, torch.full((40,), 6.0, dtype=torch.float64), 0.0, "db without a weight")
    within(dx, torch.zeros(6, 40, dtype=torch.float64), 256 * U, "dx of a sum without a weight")
    # no rows; a constant row (variance 0); leading dimensions
    e = torch.empty(0, 40, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(functional.layer_norm(e, wg, wg2 := w.clone().requires_grad_(True)), (wg, wg2),
                                 torch.empty(0, 40, device="cuda"))
    assert not dw.any() and not db.any()
    const = torch.full((3, 40), 7.25, device="cuda")
    assert torch.equal(functional.layer_norm(const, w, w), w.expand(3, 40))
    x3 = normal((2, 3, 40), 3).cuda()
    assert torch.equal(functional.layer_norm(x3, w), functional.layer_norm(x3.view(6, 40), w).view(2, 3, 40))
    # a mean that is large against the spread: the differences are taken before they are squared
    far = (normal((4, 512), 9) + 4096.0).cuda()
    ref = _ln64(far.double(), None, None, None, 1e-5).cpu()
    within(functional.layer_norm(far), ref, (512 / 8 + 16) * U * 4100.0 * 1.2, "far from 0")


def test_layer_norm_non_finite_rows_stay_alone():
    from sgnn_amd import functional
    for dtype in TYPES:
        x = normal((70, 130), 1).to(dtype).cuda()
        clean = functional.layer_norm(x)
        x[3, 7], x[9, 129] = float("nan"), float("inf")
        got = functional.layer_norm(x)
        keep = torch.ones(70, dtype=torch.bool, device="cuda")
        keep[3] = keep[9] = False
        assert torch.equal(got[keep], clean[keep]) and got[3].isnan().all() and got[9].isnan().all()


def test_layer_norm_refuses():
    from sgnn_amd import functional
    x, w = torch.zeros(3, 4, device="cuda"), torch.zeros(4, device="cuda")
    bad = [lambda: functional.layer_norm(x.double()), lambda: functional.layer_norm(x, w[:3]),
           lambda: functional.layer_norm(x, w.bfloat16()), lambda: functional.layer_norm(x.half(), w, w.half()),
           lambda: functional.layer_norm(x, w, residual=x[:2]), lambda: functional.layer_norm(x, w, eps=-1.0),
           lambda: functional.layer_norm(x, w.cpu()), lambda: functional.layer_norm(torch.zeros(3, 0, device="cuda"))]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kind", ["negated", "sparse", "expanded"])
def test_gradients_of_other_forms(kind):
    """An incoming gradient that is a lazily negated view, sparse, or one value for all."""
    from sgnn_amd import functional
    x, w, dy = normal((9, 12), 1).cuda(), normal((7, 12), 2).cuda(), normal((9, 7), 3).cuda()
    if kind == "expanded":
        dy = dy[:1, :1].expand(9, 7)
    form = {"negated": lambda t: torch._neg_view(-t), "sparse": lambda t: t.to_sparse(), "expanded": lambda t: t}[kind]
    for call in (lambda a, b: functional.linear(a, b, None, "silu"), functional.linear,
                 lambda a, b: functional.layer_norm(a[:, :7], b[:, 0])):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y = call(*leaves)
        got = torch.autograd.grad(y, leaves, form(dy), retain_graph=True)
        want = torch.autograd.grad(y, leaves, dy.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_derivatives_are_refused():
    """A dual tensor in any place, with or without a graph of the backward pass."""
    import torch.autograd.forward_ad as ad
    from sgnn_amd import functional
    t = {k: normal(s, i).cuda() for i, (k, s) in enumerate([("x", (6, 8)), ("w", (5, 8)), ("b", (5,)), ("r", (6, 5)),
                                                           ("g", (8,)), ("rx", (6, 8))])}
    with ad.dual_level():
        for k in t:
            for graph in (False, True):
                d = {n: v.clone().requires_grad_(graph) for n, v in t.items()}
                d[k] = ad.make_dual(d[k], torch.ones_like(t[k]))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad):
                        if k in "xwbr":
                            with pytest.raises(NotImplementedError, match="forward-mode"):
                                functional.linear(d["x"], d["w"], d["b"], "silu", d["r"])
                        if k in ("x", "g", "rx"):
                            with pytest.raises(NotImplementedError, match="forward-mode"):
                                functional.layer_norm(d["x"], d["g"], residual=d["rx"])


# ----------------------------------------------------------------------------- newton-schulz
def ns64(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    a, b, c = coefficients
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    norm = x.norm(dim=(-2, -1), keepdim=True) + eps
    x = torch.where(norm > 0, x / norm, torch.zeros_like(x))
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if tall else x


def ns_tol(ref, dtype, m, n):
    """Norm-wise: 15 products, each off by 4 sqrt(m + n) u of its size (rounding errors of random sign), and later
    steps' slopes multiply what came before by at most 2.2 twice (near 1, |p'(s)| / (p(s) / s) < 2.2)."""
    return 15 * 4 * (m + n) ** 0.5 * U * 2.2 ** 2 + 2 * half_step(dtype) * (dtype != torch.float32)


NS_SIZES = [(1, 1), (1, 7), (5, 1), (3, 4), (16, 16), (17, 31), (64, 64), (100, 60), (128, 128), (128, 384), (129, 200),
            (60, 515), (300, 260), (200, 1031), (128, 1024), (100, 2047), (33, 2050), (3, 4097), (520, 1100)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n", NS_SIZES)
def test_newton_schulz_against_64_bits(dtype, m, n):
    from sgnn_amd import muon
    g = (0.02 * normal((m, n), 1)).to(dtype)
    for t in (g, g.t()):
        ref = ns64(t)
        got = muon.newton_schulz(t.cuda())
        assert got.dtype == dtype and got.shape == t.shape
        err = float((got.double().cpu() - ref).norm() / ref.norm())
        assert err <= ns_tol(ref, dtype, m, n), err
    if min(m, n) >= 16:   # singular values near 1: what the steps are for
        s = torch.linalg.svdvals(muon.newton_schulz(g.cuda()).double().cpu())
        assert float(s.max()) < 1.3


@pytest.mark.parametrize("steps,coefficients", [(0, (3.4445, -4.7750, 2.0315)), (1, (1.5, -0.5, 0.0)), (12, (1.875, -1.25, 0.375))])
def test_newton_schulz_steps_and_coefficients(steps, coefficients):
    from sgnn_amd import muon
    g = normal((48, 80), 3).cuda()
    ref = ns64(g.cpu(), steps, coefficients)
    got = muon.newton_schulz(g, steps=steps, coefficients=coefficients).double().cpu()
    assert float((got - ref).norm() / ref.norm()) <= max(3 * steps, 1) * 4 * 128 ** 0.5 * U * 4
    if steps == 12:   # the cubic-order convergent polynomial: orthonormal rows
        assert float((got @ got.T - torch.eye(48, dtype=torch.float64)).abs().max()) < 1e-3


def test_newton_schulz_batches_and_lists():
    """A batch, a list of several shapes, strided and transposed inputs give each matrix' own bits."""
    from sgnn_amd import muon
    batch = normal((5, 40, 72), 1).cuda()
    alone = torch.stack([muon.newton_schulz(m) for m in batch])
    assert torch.equal(muon.newton_schulz(batch), alone)
    others = [normal((40, 72), 2).cuda(), normal((130, 150), 3).cuda(), normal((3, 20, 9), 4).cuda(), batch,
              torch.empty(0, 5, device="cuda"), normal((130, 150), 5).cuda(), normal((1, 1), 6).cuda()]
    for t, got in zip(others, muon.newton_schulz(others)):
        assert got.shape == t.shape and torch.equal(got, muon.newton_schulz(t))
    wide = normal((40, 100), 7).cuda()
    assert torch.equal(muon.newton_schulz(wide[:, 3:75]), muon.newton_schulz(wide[:, 3:75].contiguous()))
    assert torch.equal(muon.newton_schulz(wide.t()), muon.newton_schulz(wide.t().contiguous()))
    assert torch.equal(muon.newton_schulz(batch[::2]), alone[::2])
    assert torch.equal(muon.newton_schulz(batch.transpose(0, 1)[:, 1]), muon.newton_schulz(batch[1]))
    assert muon.newton_schulz([]) == []


def test_newton_schulz_by_c_with_empty_matrices():
    """Empty matrices anywhere in the array: the others, of all three kinds of launch, get the bits they get alone."""
    from sgnn_amd import _hip, muon
    shapes = [(0, 7), (4, 4), (7, 0), (64, 30), (0, 0), (128, 500), (0, 128), (300, 260), (300, 260), (0, 300), (20, 9)]
    ins = [normal(s, i).cuda() for i, s in enumerate(shapes)]
    outs = [torch.full_like(t, 9.0) for t in ins]
    mats = (_hip.SgnnMatrix * len(shapes))(*[_hip.SgnnMatrix(a.data_ptr(), b.data_ptr(), s[1], s[1], *s)
                                             for a, b, s in zip(ins, outs, shapes)])
    L = _hip.lib()
    nws = L.sgnn_newton_schulz_workspace_bytes(mats, len(shapes))
    ws = torch.empty(nws, dtype=torch.uint8, device="cuda")
    _hip.check(L.sgnn_newton_schulz(0, mats, len(shapes), 5, *muon.QUINTIC, 1e-7, ws.data_ptr(), nws,
                                    torch.cuda.current_stream().cuda_stream), "sgnn_newton_schulz")
    for a, b in zip(ins, outs):
        assert torch.equal(b, muon.newton_schulz(a))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("count,m,n", [(40, 20, 24), (70, 64, 64), (12, 128, 384), (33, 100, 300), (12, 300, 260), (9, 520, 640)])
def test_newton_schulz_of_a_batch_keeps_each_matrix_bits(dtype, count, m, n):
    from sgnn_amd import muon
    batch = (0.02 * normal((count, m, n), 1)).to(dtype).cuda()
    got = muon.newton_schulz(batch)
    for i in (0, 1, count - 1):
        assert torch.equal(got[i], muon.newton_schulz(batch[i])), i
    flipped = muon.newton_schulz(list(batch.flip(0)))
    assert all(torch.equal(a, b) for a, b in zip(flipped, got.flip(0)))
    again = batch.clone()
    assert muon.newton_schulz(again, out=again) is again and torch.equal(again, got)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("m,n", [(16, 16), (30, 64), (64, 64), (128, 384), (100, 2047), (300, 260), (520, 1100)])
def test_newton_schulz_rounds_16_bit_results_once(dtype, m, n):
    """The steps lose no more than fp32 ones, so a 16-bit result is the rounding of a y off by at most d = fp32's ns_tol.
    got is the nearest to y, so |got - y| <= |rounded(ref) - y|, and per element |got - ref| <= |got - y| + |y - ref|
    <= |rounded(ref) - ref| + 2 |y - ref|."""
    from sgnn_amd import muon
    strong = normal((m, 4), 2) @ normal((4, n), 3)   # a few strong directions: the others start far below them
    g = (0.02 * normal((m, n), 1) + 0.02 * strong).to(dtype)
    ref = ns64(g)
    once = float((ref.to(dtype).double() - ref).norm() / ref.norm())
    err = float((muon.newton_schulz(g.cuda()).double().cpu() - ref).norm() / ref.norm())
    assert err <= once + 2 * ns_tol(ref, torch.float32, m, n), (err, once)


@pytest.mark.parametrize("count,m,n", [(36, 16, 1200), (10, 224, 16), (6, 30, 900), (2, 128, 2000), (1, 520, 1100)])
def test_newton_schulz_is_as_exact_as_fp32_sums(count, m, n):
    """fp32 matrices, long sums among them: the error is at most half as large again as that of the same formula in
    fp32 products (operands have 22 bits here and 24 there; the sums must not lose more)."""
    from sgnn_amd import muon
    strong = normal((count, m, 4), 2) @ normal((count, 4, n), 3)
    g = 0.02 * normal((count, m, n), 1) + 0.02 * strong
    ref = torch.stack([ns64(t) for t in g])
    x = g.mT.contiguous() if m > n else g
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    a, b, c = muon.QUINTIC
    for _ in range(5):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    plain = x.mT if m > n else x
    err = lambda t: float((t.double().cpu() - ref).norm() / ref.norm())
    got = err(muon.newton_schulz(g.cuda()))
    print(f"fp32 {err(plain):.2e}, here {got:.2e}")
    assert got <= 1.5 * err(plain)


@pytest.mark.parametrize("m,n", [(5, 9), (128, 384), (300, 64), (100, 1500), (200, 260)])
def test_newton_schulz_without_steps_normalises(m, n):
    """x / |x| kept to 2^-21 of itself or, where it is small, 2^-34 (two fp16 planes of 2^10 x)."""
    from sgnn_amd import muon
    g = normal((m, n), 2)
    ref = ns64(g, 0)
    within(muon.newton_schulz(g.cuda(), steps=0), ref, 2.0 ** -21 * ref.abs() + 2.0 ** -34, "steps=0")


def test_newton_schulz_special_values():
    from sgnn_amd import muon
    for dtype in TYPES:
        zero = torch.zeros(30, 40, dtype=dtype, device="cuda")
        assert torch.equal(muon.newton_schulz(zero), zero) and torch.equal(muon.newton_schulz(zero, eps=0.0), zero)
        g = normal((30, 40), 1).to(dtype).cuda()
        g[4], g[:, 7] = 0, 0           # dead rows and columns stay exactly 0
        got = muon.newton_schulz(g)
        assert not got[4].any() and not got[:, 7].any()
        big = (g.float() * (2.0 ** 100 if dtype != torch.float16 else 2.0 ** 10)).to(dtype)   # squares overflow fp32
        if dtype != torch.float16:
            ref = ns64(big.cpu())
            assert float((muon.newton_schulz(big).double().cpu() - ref).norm() / ref.norm()) <= ns_tol(ref, dtype, 30, 40)
        g[0, 0] = float("nan")
        assert muon.newton_schulz(g).isnan().any()
    # tiny gradients: eps decides
    small = normal((20, 30), 2).cuda() * 1e-9
    ref = ns64(small.cpu())
    assert float((muon.newton_schulz(small).double().cpu() - ref).norm() / ref.norm()) <= ns_tol(ref, torch.float32, 20, 30)


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("m,n", [(30, 40), (128, 500), (300, 260), (2500, 20)])
def test_newton_schulz_norm_past_the_type_s_range(dtype, m, n):
    """Elements below 2^127 whose norm is above 2^128: the formula's X is an ordinary matrix."""
    from sgnn_amd import muon
    g = (normal((m, n), 1).clamp(-3.5, 3.5) * 2.0 ** 125).to(dtype)
    assert float(g.double().norm()) > 2.0 ** 128
    for steps in (0, 5):
        ref = ns64(g, steps)
        got = muon.newton_schulz(g.cuda(), steps=steps).double().cpu()
        assert float((got - ref).norm() / ref.norm()) <= ns_tol(ref, dtype, m, n), steps


def test_newton_schulz_refuses():
    from sgnn_amd import muon
    x = torch.zeros(3, 4, device="cuda")
    bad = [lambda: muon.newton_schulz(x.double()), lambda: muon.newton_schulz(x[0]), lambda: muon.newton_schulz([x, x.half()]),
           lambda: muon.newton_schulz(x, steps=-1), lambda: muon.newton_schulz(x, eps=-1.0),
           lambda: muon.newton_schulz(x[None, None]), lambda: muon.newton_schulz([x, x.cpu()]),
           lambda: muon.newton_schulz(x, out=x.t()), lambda: muon.newton_schulz(x, out=x.half()),
           lambda: muon.newton_schulz([x, x], out=[x]), lambda: muon.newton_schulz(x[None].repeat(2, 1, 1), out=x.expand(2, 3, 4)),
           lambda: muon.newton_schulz(x.to_sparse())]
    for call in bad:
        with pytest.raises(ValueError):
            call()


# ----------------------------------------------------------------------------- together
def _block(functional, x, p):
    h = functional.linear(x, p[0], p[1], "gelu")
    return functional.layer_norm(functional.linear(h, p[2], p[3], residual=x), p[4], p[5], residual=x)


def _block_params(width, hidden, dtype):
    return [normal((hidden, width), 1, width ** -0.5), normal((hidden,), 2, 0.1), normal((width, hidden), 3, hidden ** -0.5),
            normal((width,), 4, 0.1), 1.0 + normal((width,), 5, 0.1), normal((width,), 6, 0.1)]


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 4e-2)], ids=["f32", "bf16"])
def test_training_step_of_a_block(dtype, tol):
    """linear + gelu, linear + residual, layer_norm + residual, their gradients and the orthogonalised update of both
    weights, as one step: against 64 bits.  fp32: a chain of ~10 sums of <= 200 terms, (200 + 4) u * 10 < 1e-4 in the
    worst case, 1e-5 in the norm; bf16: ten roundings of 2^-9 in the norm, doubled."""
    from sgnn_amd import functional, muon
    x, dy = normal((77, 64), 11).to(dtype), normal((77, 64), 12).to(dtype)
    params = [t.to(dtype) for t in _block_params(64, 200, dtype)]
    p64 = [t.double().requires_grad_(True) for t in params]
    hid = act64(x.double() @ p64[0].T + p64[1], "gelu")
    y64 = _ln64(hid @ p64[2].T + p64[3] + x.double(), p64[4], p64[5], x.double(), 1e-5)
    g64 = torch.autograd.grad(y64, p64, dy.double())
    p = [t.cuda().requires_grad_(True) for t in params]
    y = _block(functional, x.cuda(), p)
    grads = torch.autograd.grad(y, p, dy.cuda())
    for name, got, ref in [("y", y.detach(), y64.detach())] + list(zip(["w1", "b1", "w2", "b2", "gamma", "beta"], grads, g64)):
        assert float((got.double().cpu() - ref).norm() / ref.norm()) <= tol, name
    updates = muon.newton_schulz([grads[0], grads[2]])
    for u, g in zip(updates, (grads[0], grads[2])):
        ref = ns64(g.cpu())
        assert float((u.double().cpu() - ref).norm() / ref.norm()) <= ns_tol(ref, dtype, 64, 200)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_captured_step_replays(dtype):
    """Forward, backward and the orthogonalised updates in one graph: every replay gives the eager results of the
    inputs of the moment, with eager work in between."""
    from sgnn_amd import functional, muon
    params = [t.to(dtype).cuda().requires_grad_(True) for t in _block_params(64, 200, dtype)]
    x = torch.zeros(77, 64, dtype=dtype, device="cuda")
    dy = torch.zeros(77, 64, dtype=dtype, device="cuda")

    def step():
        y = _block(functional, x, params)
        grads = torch.autograd.grad(y, params, dy)
        return [y.detach(), *grads, *muon.newton_schulz([grads[0], grads[2]])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(4):
        x.copy_(normal((77, 64), 20 + seed).to(dtype))
        dy.copy_(normal((77, 64), 30 + seed).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [o.clone() for o in outs]
        for a, b in zip(replayed, step()):
            assert torch.equal(a, b), seed


def test_two_streams_at_once():
    """The same operators on two streams, interleaved: neither sees the other's workspace."""
    from sgnn_amd import functional, muon
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    data = [[normal((2000, 96), 3 * i + j).cuda() for j in range(2)] + [normal((80, 96), 40 + i, 0.1).cuda()] for i in range(2)]

    def step(x, dy, w):
        w = w.detach().requires_grad_(True)
        y = functional.layer_norm(functional.linear(x, w, None, "silu"), None, None)
        g, = torch.autograd.grad(y, w, dy[:, :80].contiguous())
        return y.detach(), g, muon.newton_schulz(g)

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


def test_runs_repeat_bit_for_bit():
    from sgnn_amd import functional, muon
    x, dy = normal((3001, 100), 1).cuda(), normal((3001, 90), 2).cuda()
    w = normal((90, 100), 3, 0.1).cuda().requires_grad_(True)
    b, g, be = (normal((90,), i).cuda().requires_grad_(True) for i in (4, 5, 6))
    runs = []
    for _ in range(3):
        y = functional.layer_norm(functional.linear(x, w, b, "gelu"), g, be)
        grads = torch.autograd.grad(y, (w, b, g, be), dy)
        runs.append([y.detach(), *grads, muon.newton_schulz(grads[0])])
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))


# ----------------------------------------------------------------------------- the framework's paths
@pytest.mark.parametrize("dtype,activation", [(torch.float32, torch.nn.GELU), (torch.float32, torch.nn.SiLU),
                                              (torch.bfloat16, torch.nn.ReLU), (torch.float16, torch.nn.GELU)],
                         ids=["f32-gelu", "f32-silu", "bf16-relu", "f16-gelu"])
def test_modules_run_on_the_typed_operators(dtype, activation):
    """build_mlp's other activations and 16-bit parameters: an Encoder and an InteractionNetwork block, forward and
    every parameter's gradient against the same modules in float64 (norm-wise: fp32 1e-5; 16-bit types 12 roundings
    of the type along the chain)."""
    from sgnn_amd import graph_network as G
    torch.manual_seed(3)

    def mlp(i, h, o):
        return torch.nn.Sequential(G.build_mlp(i, [h], o, activation=activation), torch.nn.LayerNorm(o))
    enc, net = G.Encoder(7, 40, 3, 40, 1, 40), G.InteractionNetwork(40, 40, 40, 40, 1, 40)
    enc.node_fn, enc.edge_fn, net.node_fn, net.edge_fn = mlp(7, 40, 40), mlp(3, 40, 40), mlp(80, 40, 40), mlp(120, 40, 40)
    mods = torch.nn.ModuleList([enc, net]).to(dtype)
    ref = {k: v.detach().double().requires_grad_(True) for k, v in mods.state_dict().items()}
    mods = mods.cuda()
    n, E = 60, 300
    x, e = normal((n, 7), 1).to(dtype).float(), normal((E, 3), 2).to(dtype).float()
    ei = torch.from_numpy(np.random.default_rng(3).integers(0, n, (2, E)))
    w = normal((n, 40), 4)

    def mlp64(p, v):
        h = torch.nn.functional.linear(v, ref[p + "0.NN-0.weight"], ref[p + "0.NN-0.bias"])
        h = torch.nn.functional.linear(activation()(h), ref[p + "0.NN-1.weight"], ref[p + "0.NN-1.bias"])
        return torch.nn.functional.layer_norm(h, (h.shape[1],), ref[p + "1.weight"], ref[p + "1.bias"])
    hx, he = mlp64("0.node_fn.", x.double()), mlp64("0.edge_fn.", e.double())
    m = mlp64("1.edge_fn.", torch.cat([hx[ei[1]], hx[ei[0]], he], 1))
    want = hx + mlp64("1.node_fn.", torch.cat([torch.zeros(n, 40, dtype=torch.float64).index_add(0, ei[1], m), hx], 1))
    (want * w.double()).sum().backward()
    h0, e0 = enc(x.cuda(), e.cuda())
    got, _ = net(h0, ei.cuda(), e0)
    (got.float() * w.cuda()).sum().backward()
    h = half_step(dtype)
    tol = 1e-5 if dtype == torch.float32 else 12 * h
    got, want = got.detach(), want.detach()
    assert float((got.double().cpu() - want).norm() / want.norm()) <= tol
    if activation is torch.nn.ReLU:
        # ReLU's slope jumps: after eight roundings of h / sqrt 3 (rms) each, z is off by a relative e = h sqrt(8 / 3);
        # of two normal variables that far apart a share e / pi have different signs, and as half of the slopes are 1,
        # the dz of one layer are off by sqrt(2 e / pi) in the norm; two such layers lie on the path
        tol += (2 * 2 * h * (8 / 3) ** 0.5 / np.pi) ** 0.5
    for k, p in mods.named_parameters():
        assert float((p.grad.double().cpu() - ref[k].grad).norm() / ref[k].grad.norm()) <= tol, k


def _adam64(p, g, m, v, t, lr, b1=0.9, b2=0.999, eps=1e-8):
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


def test_muon_steps_against_64_bits():
    """Three steps on a module of several shapes (the update's formula in muon.Muon's docstring); a state_dict taken
    after two of them continues to the same bits."""
    from sgnn_amd import muon, training
    def make():
        torch.manual_seed(1)
        return torch.nn.Sequential(torch.nn.Linear(5, 40), torch.nn.Linear(40, 40), torch.nn.LayerNorm(40),
                                   torch.nn.Linear(40, 72), torch.nn.Linear(72, 3)).cuda()
    module = make()
    flat = training.FlatParams(module)
    opt = muon.Muon(flat, module, lr=0.01, weight_decay=0.1)
    params = list(module.parameters())
    matrix = [p.dim() == 2 and min(p.shape) >= 16 for p in params]
    assert sum(matrix) == 2 and opt.is_matrix == matrix
    p64 = [p.detach().double().cpu() for p in params]
    m64, v64 = [torch.zeros_like(p) for p in p64], [torch.zeros_like(p) for p in p64]
    for t in range(1, 4):
        for i, p in enumerate(params):
            g = normal(tuple(p.shape), 100 * t + i, 0.1)
            p.grad.copy_(g)
            g = g.double()
            if matrix[i]:
                m64[i] = 0.95 * m64[i] + g
                o = ns64(g + 0.95 * m64[i])
                p64[i] = p64[i] - 0.01 * (0.2 * max(p.shape) ** 0.5 * o + 0.1 * p64[i])
            else:
                p64[i], m64[i], v64[i] = _adam64(p64[i], g, m64[i], v64[i], t, 0.01)
        if t == 3:
            saved, grads = opt.state_dict(), flat.grad.clone()
            other = make()
            flat2 = training.FlatParams(other)
            flat2.param.copy_(flat.param)
            opt2 = muon.Muon(flat2, other, lr=9.0)
            opt2.load_state_dict(saved)
            flat2.grad.copy_(grads)
        opt.step()
        for i, (p, ref) in enumerate(zip(params, p64)):
            # the update's own tolerance (ns_tol at 40 + 72), on an update of lr * 0.2 * sqrt(72); Adam: a few u
            tol = ns_tol(ref, torch.float32, 40, 72) * 3 if matrix[i] else 1e-4
            assert float((p.detach().double().cpu() - ref).norm()) <= tol * (0.02 * ref.numel() ** 0.5) + 8 * U * float(ref.norm()), (t, i)
    opt2.step()
    assert torch.equal(flat2.param, flat.param)


def test_trainer_takes_muon(tmp_path):
    """Trainer(optimizer="muon") trains, checkpoints and resumes; an unknown name and another optimiser's state are
    refused."""
    from sgnn_amd import data as D, train as T
    from tests.test_gpu_harness import _config, _dataset
    md = _dataset(str(tmp_path))
    cfg = dict(_config(tmp_path), optimizer="muon")
    dev = torch.device("cuda")
    torch.manual_seed(0)
    sim = T._get_simulator(D.read_metadata(str(tmp_path)), 0.02, 0.02, dev, cfg).to(dev)
    before = {k: v.clone() for k, v in sim.state_dict().items()}
    res = T.train(sim, md, dev, cfg, log_every=1)
    assert res["step"] == 4 and all(np.isfinite(l) for _, l in res["history"])
    # (the embedding of the one particle type is not read and keeps its values)
    assert all(not torch.equal(before[k], v) for k, v in sim.state_dict().items()
               if k.endswith("weight") and "embedding" not in k)
    cfg2 = dict(cfg, model_file="model-best-000002.pt", train_state_file="train_state-best-000002.pt",
                ntraining_steps=5, nsave_steps=0)
    sim2 = T._get_simulator(md, 0.02, 0.02, dev, cfg).to(dev)
    res2 = T.train(sim2, md, dev, cfg2, log_every=1)
    assert res2["step"] == 5 and res2["trainer"].opt.step_count == 5
    with pytest.raises(ValueError, match="optimizer"):
        T.Trainer(sim2, optimizer="sgd")
    adam = T.Trainer(sim2)
    with pytest.raises(ValueError, match="Muon"):
        T.Trainer(sim2, optimizer="muon").opt.load_state_dict(adam.opt.state_dict())


def _with_activation(module, make):
    """Every ReLU of the module's MLPs replaced."""
    for m in module.modules():
        if isinstance(m, torch.nn.Sequential):
            for name, child in list(m.named_children()):
                if type(child) is torch.nn.ReLU:
                    setattr(m, name, make())
    return module


@pytest.mark.parametrize("H,nmlp,activation", [(64, 1, "gelu"), (128, 2, "silu")])
def test_simulators_and_trainers_honour_the_activation(H, nmlp, activation, monkeypatch):
    """A LearnedSimulator at the fused kernels' widths whose MLPs have another activation: one inference step and one
    Trainer step (loss and every gradient) against the oracle with that activation."""
    from oracle import sgnn_oracle as O
    from sgnn_amd.train import Trainer
    from tests.test_gpu_autograd import _check_grads, _close, _setup
    sim, osim, state, seq, types, _ = _setup(H, H, nmlp, 2)
    f = torch.nn.functional
    monkeypatch.setattr(f, "relu", getattr(f, activation))
    _with_activation(sim, {"gelu": torch.nn.GELU, "silu": torch.nn.SiLU}[activation])
    pos, nxt = torch.from_numpy(seq[:, :11]), torch.from_numpy(seq[:, 11])
    n = pos.shape[0]
    strain = torch.from_numpy(np.random.default_rng(1).normal(0, 1, n).astype(np.float32))
    noise = O.random_walk_noise(pos, 0.02, generator=torch.Generator().manual_seed(7))
    with torch.no_grad():
        want, want_strain = osim.predict_positions(pos, [n], types)
        got, got_strain = sim.predict_positions(pos.cuda(), [n], types.cuda())
        _close(got.cpu().numpy(), want.numpy(), what="positions")
        _close(got_strain.cpu().numpy(), want_strain.numpy(), what="strain")
        acc = sim.predict_accelerations(nxt.cuda(), noise.cuda(), pos.cuda(), [n], types.cuda())[0]
    pa, ta, ps = osim.predict_accelerations(nxt, noise, pos, [n], types)
    _close(acc.cpu().numpy(), pa.detach().numpy(), what="accelerations")
    with pytest.raises(NotImplementedError):
        sim.rollout_runner(pos.cuda(), [n], types.cuda(), 2)
    ref_loss = O.training_loss(pa, ta, ps, strain)
    ref_loss.backward()
    tr = Trainer(sim, lr_init=1e-3)
    out = tr.train_step(pos.cuda(), nxt.cuda(), strain.cuda(), [n], types.cuda(), noise=noise.cuda())
    assert abs(float(out["loss"]) - ref_loss.item()) <= 2e-5 * abs(ref_loss.item())
    _check_grads(sim.named_parameters(), state)


def _multi_scale(nedge_out=64):
    from oracle import multi_scale_oracle as MO
    from sgnn_amd import synthetic
    from sgnn_amd.multi_scale import MultiScaleSimulator, build_static_multi_scale_graph
    dim, T, L = 2, 6, 2
    seq = synthetic.trajectory(synthetic.lattice_2d(30, 12, x0=-1.75), T + 1, seed=13)
    st = synthetic.normalization_stats(dim, noise_std=0.02)
    stats = {k: {kk: torch.from_numpy(vv) for kk, vv in v.items()} for k, v in st.items()}
    torch.manual_seed(21)
    sim = MultiScaleSimulator(dim, (T - 1) * dim + 1, dim + 1, nedge_out, 64, L, 2, stats, 1, 9, 2, 2, 2.0)
    state = {k: v.detach().clone().requires_grad_(True) for k, v in sim.state_dict().items()}
    osim = MO.MultiScaleOracle(state, dim, L, stats, MO.create_all_edges(torch.from_numpy(seq[:, 0]), 2, 2, 2.0), 2, 2.0, 1, 2)
    sim = sim.cuda()
    sim.set_static_graph(build_static_multi_scale_graph(torch.from_numpy(seq[:, 0]).cuda(), 2, 2, 2.0))
    return sim, osim, state, torch.from_numpy(seq[:, :T]), torch.from_numpy(seq[:, T])


def test_multi_scale_simulators_and_trainers_honour_the_activation(monkeypatch):
    """The same of a MultiScaleSimulator at the fused chain's widths."""
    from oracle import sgnn_oracle as O
    from sgnn_amd.multi_scale.ms_training import MultiScaleTrainer
    from tests.test_gpu_autograd import _check_grads, _close
    sim, osim, state, pos, nxt = _multi_scale()
    monkeypatch.setattr(torch.nn.functional, "relu", torch.nn.functional.gelu)
    _with_activation(sim, torch.nn.GELU)
    n = pos.shape[0]
    strain = torch.from_numpy(np.random.default_rng(4).normal(0, 1, n).astype(np.float32))
    noise = O.random_walk_noise(pos, 0.02, generator=torch.Generator().manual_seed(5))
    pa, ta, ps = osim.predict_accelerations(nxt, noise, pos)
    with torch.no_grad():
        got = sim.predict_accelerations(nxt.cuda(), noise.cuda(), pos.cuda(), [n], None)
    _close(got[0].cpu().numpy(), pa.detach().numpy(), what="accelerations")
    _close(got[2].cpu().numpy(), ps.detach().numpy(), what="strain")
    ref_loss = O.training_loss(pa, ta, ps, strain)
    ref_loss.backward()
    tr = MultiScaleTrainer(sim, lr_init=1e-3)
    out = tr.train_step(pos.cuda(), nxt.cuda(), strain.cuda(), noise=noise.cuda())
    assert abs(float(out["loss"]) - ref_loss.item()) <= 2e-5 * abs(ref_loss.item())
    _check_grads(sim.named_parameters(), state)


def test_multi_scale_trainer_takes_muon():
    """MultiScaleTrainer(optimizer="muon"): its step is Muon's on the gradient that it formed."""
    from sgnn_amd import muon, training
    from sgnn_amd.multi_scale.ms_training import MultiScaleTrainer
    (sim, _, _, pos, nxt), (other, *_) = _multi_scale(), _multi_scale()
    tr = MultiScaleTrainer(sim, lr_init=1e-3, optimizer="muon")
    assert tr.fused and sum(tr.opt.is_matrix) > 10
    flat = training.FlatParams(other)
    opt = muon.Muon(flat, other, 1e-3)
    for _ in range(2):
        opt.lr = tr.opt.lr   # the schedule sets the next step's after each
        tr.train_step(pos.cuda(), nxt.cuda(), torch.zeros(pos.shape[0], device="cuda"))
        flat.grad.copy_(tr.flat.grad)
        before = flat.param.clone()
        opt.step()
        assert torch.equal(flat.param, tr.flat.param) and not torch.equal(flat.param, before)


def test_activations_of_derived_classes_and_unknown_ones():
    """A class derived from nn.GELU is GELU (it got ReLU); an activation that no kernel computes is refused everywhere,
    and so is one where the ReLU kernels have none."""
    from sgnn_amd import graph_network as G

    class Named(torch.nn.GELU):
        pass

    x, e = normal((20, 7), 1).cuda(), normal((30, 3), 2).cuda()
    outs = []
    for make in (torch.nn.GELU, Named):
        torch.manual_seed(5)
        outs.append(_with_activation(G.Encoder(7, 40, 3, 40, 1, 40).cuda(), make)(x, e))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    with pytest.raises(NotImplementedError, match="Tanh"):
        _with_activation(G.Encoder(7, 40, 3, 40, 1, 40).cuda(), torch.nn.Tanh)(x, e)
    ei = torch.zeros(2, 30, dtype=torch.int64, device="cuda")
    epd = _with_activation(G.EncodeProcessDecode(7, 3, 3, 64, 2, 1, 64).cuda(), torch.nn.Tanh)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="Tanh"):
        epd(x, ei, e)
    # an output activation
    dec = G.Decoder(40, 3, 1, 40).cuda()
    dec.node_fn = G.build_mlp(40, [40], 3, output_activation=torch.nn.ReLU).cuda()
    h = normal((50, 40), 3).cuda()
    got = dec(h)
    p = dict(dec.node_fn.named_parameters())
    ref = torch.relu(torch.relu(h.double() @ p["NN-0.weight"].double().T + p["NN-0.bias"].double()) @ p["NN-1.weight"].double().T
                     + p["NN-1.bias"].double())
    within(got, ref.detach().cpu(), 84 * U * 40, "output activation")   # sums of 40 products of magnitude < 1


def test_simulators_with_16_bit_parameters():
    """A bf16 simulator at the fused kernels' widths computes in bf16 and returns fp32 (26 roundings of the type along the
    chain: encoder 3, three blocks of 7, decoder 2); a Trainer makes its parameters fp32 and takes the fused kernels."""
    from oracle import sgnn_oracle as O
    from sgnn_amd.train import Trainer
    from tests.test_gpu_autograd import _setup
    sim, osim, state, seq, types, _ = _setup(64, 64, 1, 2)
    sim = sim.bfloat16()
    with torch.no_grad():
        for v in state.values():
            v.copy_(v.bfloat16().float())
        pos, nxt = torch.from_numpy(seq[:, :11]), torch.from_numpy(seq[:, 11])
        n = pos.shape[0]
        zero = torch.zeros_like(pos)
        want = osim.predict_accelerations(nxt, zero, pos, [n], types)
        got = sim.predict_accelerations(nxt.cuda(), zero.cuda(), pos.cuda(), [n], types.cuda())
        for a, b in ((got[0], want[0]), (got[2], want[2])):
            assert a.dtype == torch.float32
            assert float((a.cpu() - b).norm() / b.norm()) <= 26 * half_step(torch.bfloat16)
        assert sim.predict_positions(pos.cuda(), [n], types.cuda())[0].dtype == torch.float32
    tr = Trainer(sim, lr_init=1e-3)
    assert tr.fused and all(p.dtype == torch.float32 for p in sim.parameters())
    pa, ta, ps = osim.predict_accelerations(nxt, zero, pos, [n], types)
    strain = torch.zeros(n)
    out = tr.train_step(pos.cuda(), nxt.cuda(), strain.cuda(), [n], types.cuda(), noise=zero.cuda())
    ref = O.training_loss(pa, ta, ps, strain)
    assert abs(float(out["loss"]) - ref.item()) <= 2e-5 * abs(ref.item())
