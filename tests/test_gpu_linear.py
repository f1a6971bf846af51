"""The dense layer with its fused epilogue (ccn_linear_*) and its gradients (ccn_linear_backward_*) against a float64
restatement of the formulas.

Tolerances are sums of what each rounding may add, for element y with S = sum |x||w| (+ |bias|):
  - the product: an fp32 sum of T terms in any order, T * 2^-24 * S (products of 16-bit operands are exact in fp32);
  - an activation or its slope in fp32: 2^-20 of its argument's scale (all slopes used here are below 1.2);
  - a rounding to 16 bits: eps/2 relative (bf16 2^-8, fp16 2^-11, and 2^-25 absolute among fp16's subnormals);
  - dz, rounded to 16 bits before the two products when there is an activation, carries that half step times |w| or |x|.
Inputs lie in rows with padding that holds NaN, outputs in buffers that hold a marker: neither may show up or vanish.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
TYPES = {False: torch.bfloat16, True: torch.float16}
U24 = 2.0 ** -24
FN = 2.0 ** -20          # an activation or slope in fp32
MARK = 7.0


def half_step(half):
    return 2.0 ** -11 if half else 2.0 ** -8


def tiny(half):
    return 2.0 ** -25 if half else 2.0 ** -126


def matrix(gen, rows, cols, half, scale=1.0, pad=0, shift=0):
    """[rows x cols] inside rows of cols + pad elements whose padding is NaN, `shift` elements into the allocation."""
    buf = torch.full((shift + rows * (cols + pad) + 8,), math.nan, device=DEV, dtype=TYPES[half])
    view = buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_(torch.randn(rows, cols, device=DEV, generator=gen) * scale)
    return view


class Out:
    """An output matrix in a buffer of markers."""

    def __init__(self, rows, cols, dtype, pad=0, shift=0):
        self.buf = torch.full((shift + rows * (cols + pad) + 16,), MARK, device=DEV, dtype=dtype)
        self.view = self.buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]

    def outside_is_untouched(self):
        keep = self.view.clone()
        self.view.fill_(MARK)
        ok = bool((self.buf == MARK).all())
        self.view.copy_(keep)
        return ok


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    z = z.clone().requires_grad_(True)
    if act == "relu":
        return (z.detach() > 0).double()
    y = act64(z, act)
    return torch.autograd.grad(y.sum(), z)[0]


def within(got, want, tol, what):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    d = (got.double() - want).abs()
    worst = (d / tol).max().item() if d.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def forward_case(ccn, M, N, K, act, half, bias=True, resid=True, keep=True, pad=0, shift=0, seed=0, plan=None, stream=None):
    g = gen(seed + M * 7 + N * 11 + K * 13)
    X, W = matrix(g, M, K, half, 1.0, pad, shift), matrix(g, K, N, half, 1.0 / math.sqrt(K), pad, shift)
    R = matrix(g, M, N, half, 1.0, pad, shift) if resid else None
    b = torch.randn(N + 1, device=DEV, generator=g)[1:] if bias else None   # fp32, 4-byte aligned only
    Y, P = Out(M, N, TYPES[half], pad, shift), (Out(M, N, TYPES[half], pad, shift) if keep else None)
    own = plan or ccn.LinearPlan(M, N, K)
    own.forward(X, W, b, R, Y.view, M, N, K, act=act, pre=P.view if keep else None, half=half, ldx=K + pad, ldw=N + pad, ldr=N + pad,
                ldy=N + pad, ldp=N + pad, stream=stream)
    torch.cuda.synchronize()
    x, w = X.double(), W.double()
    z, S = x @ w, x.abs() @ w.abs()
    if bias:
        z, S = z + b.double(), S + b.double().abs()
    y = act64(z, act)
    y = y + R.double() if resid else y
    h = half_step(half)
    base = (K + 2) * U24 * S
    tol = 1.2 * base + FN * (z.abs() + 1) + 2 * U24 * y.abs() + (1 + 2 * h) * h * (y.abs() + 1.2 * base) + tiny(half)
    within(Y.view, y, tol, f"Y {M}x{N}x{K} {act}")
    assert Y.outside_is_untouched()
    if keep:
        within(P.view, z, base + (1 + 2 * h) * h * (z.abs() + base) + tiny(half), f"pre {M}x{N}x{K}")
        assert P.outside_is_untouched()
    if plan is None:
        own.close()


SHAPES = [(1, 1, 1), (1, 8, 8), (1, 64, 1024), (1, 8192, 1024), (2, 257, 63), (3, 130, 4099), (5, 2049, 515), (15, 1000, 333), (16, 4096, 2048), (17, 72, 4096),
          (31, 777, 129), (32, 512, 64), (33, 520, 1030), (48, 1024, 4096), (64, 640, 8192), (65, 128, 64), (127, 129, 65), (128, 128, 128), (129, 255, 1),
          (3, 1000, 130), (4, 33, 2047), (4, 7, 5), (100, 5, 300), (100, 300, 5), (300, 3, 5), (70, 7, 200),
          (255, 256, 32), (256, 264, 40), (300, 301, 302), (512, 512, 1024), (777, 1025, 513), (1000, 2056, 1032), (2048, 1024, 96)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("half", [False, True], ids=["bf16", "f16"])
def test_forward_shapes(ccn, M, N, K, half):
    i = SHAPES.index((M, N, K))
    forward_case(ccn, M, N, K, ACTS[i % 5], half, bias=i % 3 != 0, resid=i % 2 == 0, keep=i % 4 < 2)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(4, 200, 136), (70, 200, 136), (600, 520, 264)])
def test_forward_activations(ccn, M, N, K, act):
    for half in (False, True):
        for bias, resid, keep in ((True, True, True), (False, False, False), (True, False, True), (False, True, False)):
            forward_case(ccn, M, N, K, act, half, bias, resid, keep)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 5), (8, 0), (8, 8), (64, 4)])
@pytest.mark.parametrize("M,N,K", [(1, 136, 264), (13, 1001, 520), (64, 128, 128), (200, 131, 135), (384, 512, 256)])
def test_forward_strides_and_alignments(ccn, M, N, K, pad, shift):
    forward_case(ccn, M, N, K, "silu", False, pad=pad, shift=shift)
    forward_case(ccn, M, N, K, "gelu", True, pad=pad, shift=shift)


@pytest.mark.parametrize("M,N,K,half", [(4096, 4096, 256, False), (4096, 4104, 136, True), (4100, 4096, 520, False), (8192, 2048, 1024, False), (3000, 6000, 1000, True),
                                         (2048, 4096, 1024, False), (2040, 4000, 1000, True), (2000, 4001, 1003, False),
                                         (16, 8200, 6200, False), (40, 8193, 6203, True), (5, 6211, 8200, False)])
def test_forward_large(ccn, M, N, K, half):
    forward_case(ccn, M, N, K, "gelu_tanh", half, resid=True, keep=True)


def test_forward_extreme_values(ccn):
    """Pre-activations far out on both sides: the activations are 0 or z there (|silu(-90)| = 90 e^-90 < 1e-37, its slope
    less than that again), and nothing becomes NaN."""
    M, N, K = 4, 64, 8
    X = torch.zeros(M, K, device=DEV, dtype=torch.bfloat16)
    X[:, 0] = 1.0
    W = torch.zeros(K, N, device=DEV, dtype=torch.bfloat16)
    W[0] = torch.tensor([1e30, -1e30, 1e4, -1e4, 200.0, -200.0, 90.0, -90.0] * 8, device=DEV)
    plan = ccn.LinearPlan(M, N, K)
    for act in ACTS:
        Y = torch.empty(M, N, device=DEV, dtype=torch.bfloat16)
        plan.forward(X, W, None, None, Y, M, N, K, act=act)
        z = W[0].double()
        want = z if act == "none" else torch.where(z > 0, z, torch.zeros_like(z))
        assert (Y.double() - want.expand(M, N).to(torch.bfloat16).double()).abs().max() <= 1e-36, act
        pre = W[0].expand(M, N).contiguous()
        dY = torch.ones(M, N, device=DEV, dtype=torch.bfloat16)
        db = torch.empty(N, device=DEV)
        plan.backward(dY, pre, None, None, None, None, db, M, N, K, act=act)
        slope = torch.ones_like(z) if act == "none" else (z > 0).double()
        assert (db.double() - slope * M).abs().max() <= 1e-36, act
    plan.close()


def test_forward_infinities_and_nan_stay_in_their_row(ccn):
    """A row of X that holds inf or NaN spoils that row of Y only, whatever the tile edges."""
    for M, N, K in ((3, 40, 70), (130, 200, 100), (300, 264, 72)):
        g = gen(M)
        X, W = matrix(g, M, K, False), matrix(g, K, N, False)
        clean, dirty = (torch.empty(M, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        plan = ccn.LinearPlan(M, N, K)
        plan.forward(X, W, None, None, clean, M, N, K)
        X = X.clone()
        X[1, K - 1] = math.inf
        X[M - 1, 0] = math.nan
        plan.forward(X, W, None, None, dirty, M, N, K)
        rows = torch.ones(M, dtype=torch.bool, device=DEV)
        rows[1] = rows[M - 1] = False
        assert torch.equal(clean[rows], dirty[rows])
        assert not torch.isfinite(dirty[1]).any() and torch.isnan(dirty[M - 1]).all()
        plan.close()


def backward_case(ccn, M, N, K, act, half, dw32=False, accumulate=False, pad=0, shift=0, want=("dX", "dW", "db"), seed=0):
    g = gen(seed + M * 5 + N * 3 + K)
    t = TYPES[half]
    dY, X, W = matrix(g, M, N, half, 1.0, pad, shift), matrix(g, M, K, half, 1.0, pad, shift), matrix(g, K, N, half, 0.1, pad, shift)
    pre = matrix(g, M, N, half, 1.5, pad, shift) if act != "none" else None
    dX, dW = Out(M, K, t, pad, shift), Out(K, N, torch.float32 if dw32 else t, pad, shift)
    db = Out(1, N, torch.float32, 0, 1)
    if accumulate:
        dW.view.normal_(generator=g)
        db.view.normal_(generator=g)
    dW0, db0 = dW.view.double().clone(), db.view[0].double().clone()
    plan = ccn.LinearPlan(M, N, K)
    plan.backward(dY, pre, X if "dW" in want else None, W if "dX" in want else None, dX.view if "dX" in want else None, dW.view if "dW" in want else None,
                  db.view if "db" in want else None, M, N, K, act=act, half=half, dw_f32=dw32, accumulate=accumulate, lddy=N + pad, ldp=N + pad,
                  ldx=K + pad, ldw=N + pad, lddx=K + pad, lddw=N + pad)
    torch.cuda.synchronize()
    h = half_step(half)
    dy, x, w = dY.double(), X.double(), W.double()
    dz, e = dy, torch.zeros_like(dy)      # e: what the rounded dz may be off by
    if act != "none":
        dz = dy * slope64(pre.double(), act)
        e = (1 + h) * h * dz.abs() + FN * dy.abs() * (1.0 + pre.double().abs()) + tiny(half)
    if "dX" in want:
        v = dz @ w.t()
        base = N * U24 * ((dz.abs() + e) @ w.abs().t()) + e @ w.abs().t()
        within(dX.view, v, base + (1 + 2 * h) * h * (v.abs() + base) + tiny(half), f"dX {M}x{N}x{K} {act}")
        assert dX.outside_is_untouched()
    else:
        assert bool((dX.buf == MARK).all())
    if "dW" in want:
        v = x.t() @ dz
        base = (M + 2) * U24 * (x.abs().t() @ (dz.abs() + e)) + x.abs().t() @ e
        if accumulate:
            v = v + dW0
            base = base + 2 * U24 * (v.abs() + dW0.abs())
        tol = base + 2 * U24 * v.abs() + 1e-38 if dw32 else base + (1 + 2 * h) * h * (v.abs() + base) + tiny(half)
        within(dW.view, v, tol, f"dW {M}x{N}x{K} {act}")
        assert dW.outside_is_untouched()
    else:
        assert bool((dW.buf == MARK).all())
    if "db" in want:
        v = dz.sum(0)
        base = (M + 2) * U24 * dz.abs().sum(0)
        if act != "none":
            base = base + (FN * dy.abs() * (1.0 + pre.double().abs())).sum(0)
        if accumulate:
            v = v + db0
            base = base + 2 * U24 * (v.abs() + db0.abs())
        within(db.view[0], v, base + 1e-38, f"db {M}x{N}x{K} {act}")
        assert db.outside_is_untouched()
    plan.close()


BSHAPES = [(1, 1, 1), (1, 64, 128), (2, 513, 70), (7, 130, 1031), (16, 1024, 512), (33, 65, 129), (64, 256, 256), (128, 128, 128), (130, 257, 131), (255, 1000, 72),
           (256, 512, 1024), (515, 264, 2049), (1001, 515, 1025), (2048, 256, 256), (4097, 136, 200),
           (300, 3, 5), (100, 5, 300), (500, 300, 5), (1000, 6, 40), (20, 2100, 2060), (190, 2100, 2053),
           (4500, 120, 264), (3000, 301, 100), (300, 3000, 296), (257, 2999, 131)]


@pytest.mark.parametrize("M,N,K", BSHAPES)
@pytest.mark.parametrize("half", [False, True], ids=["bf16", "f16"])
def test_backward_shapes(ccn, M, N, K, half):
    i = BSHAPES.index((M, N, K))
    backward_case(ccn, M, N, K, ACTS[i % 5], half)
    backward_case(ccn, M, N, K, "none", half, dw32=True, accumulate=i % 2 == 0)


@pytest.mark.parametrize("act", ACTS)
def test_backward_activations(ccn, act):
    for half in (False, True):
        backward_case(ccn, 200, 136, 264, act, half)
        backward_case(ccn, 200, 136, 264, act, half, dw32=True)
        backward_case(ccn, 200, 136, 264, act, half, dw32=True, accumulate=True)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 5), (8, 8)])
@pytest.mark.parametrize("M,N,K", [(9, 137, 65), (256, 256, 256), (300, 129, 520)])
def test_backward_strides_and_alignments(ccn, M, N, K, pad, shift):
    backward_case(ccn, M, N, K, "gelu_tanh", False, pad=pad, shift=shift)
    backward_case(ccn, M, N, K, "none", True, dw32=True, accumulate=True, pad=pad, shift=shift)


@pytest.mark.parametrize("want", [("dX",), ("dW",), ("db",), ("dX", "db"), ("dW", "db"), ("dX", "dW")], ids="+".join)
def test_backward_parts(ccn, want):
    backward_case(ccn, 150, 264, 136, "silu", False, want=want)
    backward_case(ccn, 150, 264, 136, "none", False, want=want)


@pytest.mark.parametrize("M,N,K,act,half", [(4096, 4096, 4096, "gelu", False), (8192, 2048, 2056, "none", False), (4100, 4104, 4096, "relu", True),
                                              (1024, 4096, 2048, "none", False), (1000, 4090, 2040, "none", True), (1000, 4001, 2003, "silu", False)])
def test_backward_large(ccn, M, N, K, act, half):
    backward_case(ccn, M, N, K, act, half, dw32=act == "none")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_backward_against_differences(ccn, act):
    """The gradients along random directions against central differences of the loss sum(Y * G), computed in float64 from
    the same 16-bit inputs.  The difference itself is off by O(step^2); the gradients by their bf16 roundings, whose
    errors add up at random along a direction: 6 sigma of a half step's uniform error per element."""
    M, N, K = 96, 72, 56
    g = gen(11)
    X, W, G = matrix(g, M, K, False), matrix(g, K, N, False, 0.2), matrix(g, M, N, False)
    pre, Y = (torch.empty(M, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    dX, dW, db = torch.empty(M, K, device=DEV, dtype=torch.bfloat16), torch.empty(K, N, device=DEV), torch.empty(N, device=DEV)
    b = torch.randn(N, device=DEV, generator=g)
    plan = ccn.LinearPlan(M, N, K)
    plan.forward(X, W, b, None, Y, M, N, K, act=act, pre=pre)
    plan.backward(G, pre, X, W, dX, dW, db, M, N, K, act=act, dw_f32=True)
    x, w, bb, gg = X.double(), W.double(), b.double(), G.double()
    loss = lambda x, w, bb: (act64(x @ w + bb, act) * gg).sum()  # noqa: E731
    h = 1e-5
    h8 = 2.0 ** -8
    dz = gg * slope64(pre.double(), act)
    # pre is rounded to bf16 too: its half step moves the slope by at most that times |act''| <= 1.2
    e = h8 * (dz.abs() + 1.2 * gg.abs() * pre.double().abs())
    for seed in range(4):
        gd = gen(seed)
        for name, grad, at, err in (("X", dX, x, (e.square() @ w.t().square() + (h8 * dX.double()).square())), ("W", dW, w, x.t().square() @ e.square()),
                                    ("b", db, bb, e.square().sum(0))):
            d = torch.randn(at.shape, device=DEV, generator=gd, dtype=torch.float64)
            args = {"X": x, "W": w, "b": bb}
            up, down = dict(args), dict(args)
            up[name], down[name] = at + h * d, at - h * d
            diff = (loss(up["X"], up["W"], up["b"]) - loss(down["X"], down["W"], down["b"])) / (2 * h)
            got = (grad.double() * d).sum()
            tol = 6 * (err * d.square()).sum().sqrt() + 1e-6 * abs(diff)
            assert abs(got - diff) <= tol, (name, got.item(), diff.item(), tol.item())
    plan.close()


def test_empty_batch(ccn):
    plan = ccn.LinearPlan(8, 64, 32)
    dW, db = torch.full((32, 64), 3.0, device=DEV), torch.full((64,), 3.0, device=DEV)
    plan.forward(None, None, None, None, None, 0, 64, 32, act="relu")
    plan.backward(None, None, None, None, None, dW, db, 0, 64, 32, act="relu", dw_f32=True, accumulate=True)
    assert bool((dW == 3).all()) and bool((db == 3).all())
    plan.backward(None, None, None, None, None, dW, db, 0, 64, 32, act="relu", dw_f32=True)
    assert not dW.any() and not db.any()
    dW16 = torch.full((32, 64), 3.0, device=DEV, dtype=torch.bfloat16)
    plan.backward(None, None, None, None, None, dW16, None, 0, 64, 32)
    assert not dW16.any()
    plan.close()


@pytest.mark.parametrize("M,N,K", [(2112, 136, 200), (40, 136, 2112), (3, 136, 2048), (2100, 129, 201)])
def test_rows_far_apart(ccn, M, N, K):
    """Rows 2^21 elements apart: offsets inside the matrices pass 2^32, inside a tile 2^30."""
    g, ld, rows = gen(M), 1 << 21, max(M, K)
    big = [torch.empty(rows * ld, device=DEV, dtype=torch.bfloat16) for _ in range(4)]
    far = [b.view(rows, ld) for b in big]
    X, W, G, R = matrix(g, M, K, False), matrix(g, K, N, False, 0.1), matrix(g, M, N, False), matrix(g, M, N, False)
    b = torch.randn(N, device=DEV, generator=g)
    plan = ccn.LinearPlan(M, N, K)
    y, pre = (torch.empty(M, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    dx, dw, db, db2 = torch.empty_like(X, memory_format=torch.contiguous_format), torch.empty(K, N, device=DEV, dtype=torch.bfloat16), torch.empty(N, device=DEV), torch.empty(N, device=DEV)
    plan.forward(X, W, b, R, y, M, N, K, act="silu", pre=pre)
    plan.backward(G, pre, X, W, dx, dw, db, M, N, K, act="silu")
    x2, w2, y2, p2 = far[0][:M, :K], far[1][:K, :N], far[2][:M, :N], far[3][:M, :N]
    x2.copy_(X), w2.copy_(W), y2.copy_(R)
    plan.forward(x2, w2, b, y2, y2, M, N, K, act="silu", pre=p2, ldx=ld, ldw=ld, ldr=ld, ldy=ld, ldp=ld)
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(pre, p2)
    g2, dx2, dw2 = far[2][:M, 4096:4096 + N], far[2][:M, 8192:8192 + K], far[3][:K, 8192:8192 + N]
    g2.copy_(G)
    plan.backward(g2, p2, x2, w2, dx2, dw2, db2, M, N, K, act="silu", lddy=ld, ldp=ld, ldx=ld, ldw=ld, lddx=ld, lddw=ld)
    torch.cuda.synchronize()
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)
    plan.close()


def test_residual_in_place(ccn):
    """Y may be the residual itself."""
    for M, N, K in ((1, 200, 300), (40, 1024, 512), (300, 264, 100), (512, 4096, 128)):
        g = gen(M)
        X, W, R = matrix(g, M, K, False), matrix(g, K, N, False, 0.05), matrix(g, M, N, False)
        Y = torch.empty(M, N, device=DEV, dtype=torch.bfloat16)
        plan = ccn.LinearPlan(M, N, K)
        plan.forward(X, W, None, R, Y, M, N, K, act="silu")
        Z = R.clone()
        plan.forward(X, W, None, Z, Z, M, N, K, act="silu")
        assert torch.equal(Y, Z)
        plan.close()


def test_one_plan_many_sizes_and_same_bits(ccn):
    """A plan of the largest size serves smaller calls, back to back and in any order; the same call gives the same bits."""
    plan = ccn.LinearPlan(600, 1100, 1300)
    for M, N, K in ((600, 1100, 1300), (1, 1100, 1300), (64, 1100, 1300), (600, 8, 1300), (1, 1, 1), (17, 1029, 1300), (600, 1100, 8)):
        forward_case(ccn, M, N, K, "gelu", False, plan=plan)
        g = gen(1)
        X, W = matrix(g, M, K, False), matrix(g, K, N, False)
        a, b = (torch.empty(M, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        plan.forward(X, W, None, None, a, M, N, K)
        plan.forward(X, W, None, None, b, M, N, K)
        assert torch.equal(a, b)
    plan.close()


def test_streams_and_recording(ccn):
    """Forward and backward on a stream of the library's own, then recorded and replayed with new inputs in the same buffers,
    with eager calls between the replays."""
    for M, N, K in ((1, 512, 2048), (48, 264, 1024), (300, 520, 264)):
        g = gen(M)
        plan, st = ccn.LinearPlan(M, N, K), ccn.Stream()
        X, W, b, G = matrix(g, M, K, False), matrix(g, K, N, False, 0.05), torch.randn(N, device=DEV, generator=g), matrix(g, M, N, False)
        outs = [torch.empty(M, N, device=DEV, dtype=torch.bfloat16), torch.empty(M, N, device=DEV, dtype=torch.bfloat16),
                torch.empty(M, K, device=DEV, dtype=torch.bfloat16), torch.empty(K, N, device=DEV), torch.empty(N, device=DEV)]

        def calls(stream, o):
            plan.forward(X, W, b, None, o[0], M, N, K, act="gelu", pre=o[1], stream=stream)
            plan.backward(G, o[1], X, W, o[2], o[3], o[4], M, N, K, act="gelu", dw_f32=True, stream=stream)

        torch.cuda.synchronize()
        graph = ccn.Graph(st)
        with graph:
            calls(st.h, outs)
        for rep in range(3):
            X.normal_(generator=g)
            G.normal_(generator=g)
            torch.cuda.synchronize()
            graph.launch()
            st.sync()
            eager = [torch.empty_like(o) for o in outs]
            calls(None, eager)
            torch.cuda.synchronize()
            for a, e in zip(outs, eager):
                assert torch.equal(a, e), rep
        graph.close()
        plan.close()
        st.close()


def test_refusals(ccn):
    plan = ccn.LinearPlan(64, 128, 256)
    X, W = torch.zeros(64, 256, device=DEV, dtype=torch.bfloat16), torch.zeros(256, 128, device=DEV, dtype=torch.bfloat16)
    Y, b = torch.full((64, 128), 5.0, device=DEV, dtype=torch.bfloat16), torch.zeros(128, device=DEV)
    dW = torch.full((256, 128), 5.0, device=DEV, dtype=torch.bfloat16)
    dX = torch.full((64, 256), 5.0, device=DEV, dtype=torch.bfloat16)
    E, R = ccn.CCN_EINVAL, ccn.CCN_ERANGE

    def refused(code, f, *a, **k):
        with pytest.raises(ccn.CoconetError) as e:
            f(*a, **k)
        assert e.value.code == code

    f, bw = plan.forward, plan.backward
    refused(E, f, None, W, b, None, Y, 64, 128, 256)
    refused(E, f, X, None, b, None, Y, 64, 128, 256)
    refused(E, f, X, W, b, None, None, 64, 128, 256)
    refused(E, f, X.data_ptr() + 1, W, b, None, Y, 64, 128, 256)
    refused(E, f, X, W, b.data_ptr() + 2, None, Y, 64, 128, 256)
    refused(E, f, X, W, b, None, Y, 64, 128, 256, ldx=255)
    refused(E, f, X, W, b, None, Y, 64, 128, 256, ldy=127)
    refused(E, f, X, W, b, Y, Y, 64, 128, 256, ldr=127)
    refused(R, f, X, W, b, None, Y, 64, 128, 256, ldx=(1 << 22) + 1)
    refused(R, f, X, W, b, None, Y, 65, 128, 256)
    refused(R, f, X, W, b, None, Y, 64, 129, 256)
    refused(R, f, X, W, b, None, Y, 64, 128, 257)
    refused(E, f, X, W, b, None, Y, -1, 128, 256)
    refused(E, f, X, W, b, None, Y, 64, 0, 256)
    refused(E, f, X, W, b, None, Y, 64, 128, 0)
    refused(E, bw, Y, None, X, W, dX, dW, b, 64, 128, 256, act="gelu")            # an activation without pre
    refused(E, bw, Y, None, X, None, dX, dW, b, 64, 128, 256)                     # dX without W
    refused(E, bw, Y, None, None, W, dX, dW, b, 64, 128, 256)                     # dW without X
    refused(E, bw, Y, None, X, W, dX, dW, b, 64, 128, 256, accumulate=True)       # a 16-bit dW is not added to
    refused(E, bw, None, None, X, W, dX, dW, b, 64, 128, 256)
    refused(E, bw, Y, None, X, W, dX, dW, b, 64, 128, 256, lddw=100)
    lib = ccn.load()
    bad = (plan.h, X.data_ptr(), 256, W.data_ptr(), 128, None, None, 0, Y.data_ptr(), 128, None, 0, 64, 128, 256)
    assert lib.ccn_linear_bf16(*bad, 5, None) == E and lib.ccn_linear_bf16(*bad, -1, None) == E
    assert lib.ccn_linear_backward_bf16(plan.h, Y.data_ptr(), 128, None, 0, X.data_ptr(), 256, W.data_ptr(), 128, dX.data_ptr(), 256, dW.data_ptr(), 128, 2, None, 0,
                                        64, 128, 256, 0, None) == E               # an f16 dW of a bf16 layer
    torch.cuda.synchronize()
    assert bool((Y == 5).all()) and bool((dW == 5).all()) and bool((dX == 5).all())
    plan.close()


@pytest.mark.parametrize("half", [False, True], ids=["bf16", "f16"])
@pytest.mark.parametrize("M", [2, 20, 70])
def test_gelu_far_left(ccn, M, half):
    """GELU and its slope where both are a small tail: within 2^-18 relative (the fit, a dozen fp32 roundings, exp2 and the reciprocal at 1
    ulp) and the exponent's roundings (four of 2^-24 of z^2/2), beside the output's own half step."""
    N, K = 1400, 8
    X = torch.zeros(M, K, device=DEV, dtype=TYPES[half])
    X[:, 0] = 1.0
    W = torch.zeros(K, N, device=DEV, dtype=TYPES[half])
    W[0] = torch.linspace(-10.0, -3.0, N, device=DEV)
    z = W[0].double()
    phi, Phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), torch.erfc(-z * math.sqrt(0.5)) / 2   # (ndtr on the device is 0 below -8)
    rel = 2.0 ** -18 + 4 * U24 * z * z / 2
    Y = torch.empty(M, N, device=DEV, dtype=TYPES[half])
    plan = ccn.LinearPlan(M, N, K)
    plan.forward(X, W, None, None, Y, M, N, K, act="gelu", half=half)
    y = (z * Phi).expand(M, N)
    h = half_step(half)
    within(Y, y, (h + (1 + h) * rel) * y.abs() + tiny(half), f"Y {M}")
    pre, dY, db = W[0].expand(M, N).contiguous(), torch.ones(M, N, device=DEV, dtype=TYPES[half]), torch.empty(N, device=DEV)
    plan.backward(dY, pre, None, None, None, None, db, M, N, K, act="gelu", half=half)
    s = M * (Phi + z * phi)
    within(db, s, M * (rel + (M + 2) * U24) * (Phi + z.abs() * phi), f"db {M}")
    plan.close()


def test_tensors_that_are_not_what_they_are_taken_for(ccn):
    """Types, devices and orders of the Python call's tensors: refused before anything is launched.  What lies as the call
    reads it is taken, however it is shaped."""
    M, N, K = 6, 16, 24
    g = gen(1)
    X, W, b = matrix(g, M, K, False), matrix(g, K, N, False), torch.randn(N, device=DEV, generator=g)
    Y, dW, db = torch.full((M, N), 5.0, device=DEV, dtype=torch.bfloat16), torch.full((K, N), 5.0, device=DEV), torch.full((N,), 5.0, device=DEV)
    dX = torch.full((M, K), 5.0, device=DEV, dtype=torch.bfloat16)
    plan = ccn.LinearPlan(2 * M, N, K)
    E, R = ccn.CCN_EINVAL, ccn.CCN_ERANGE

    def refused(code, f, *a, **k):
        with pytest.raises(ccn.CoconetError) as e:
            f(*a, **k)
        assert e.value.code == code

    for X2, W2, b2, Y2 in ((X.float(), W, b, Y), (X.half(), W, b, Y), (X.cpu(), W, b, Y), (X, W.t().contiguous().t(), b, Y), (X, W, b.bfloat16(), Y),
                           (X, W, b, Y.float()), (torch.cat([X, X], 1)[:, :K], W, b, Y)):
        refused(E, plan.forward, X2, W2, b2, None, Y2, M, N, K)
    refused(R, plan.forward, X, W, b[:8], None, Y, M, N, K)
    refused(E, plan.forward, X, W, b, Y.half(), Y, M, N, K)
    refused(E, plan.forward, X, W, b, None, Y, M, N, K, pre=Y.float())
    refused(E, plan.forward, X, W, b, None, Y, M, N, K, half=True)
    refused(E, plan.backward, Y, None, X, W, dX, dW, db, M, N, K)                       # an fp32 dW without dw_f32
    refused(E, plan.backward, Y, None, X, W, dX, dW.bfloat16(), db, M, N, K, dw_f32=True)
    refused(E, plan.backward, Y, X.float(), X, W, dX, dW, db, M, N, K, act="silu", dw_f32=True)
    refused(E, plan.backward, Y, None, X, W, dX.t().contiguous().t(), dW, db, M, N, K, dw_f32=True)
    torch.cuda.synchronize()
    assert all(bool((x == 5).all()) for x in (Y, dW, db, dX))
    want, got = (torch.empty(M, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    plan.forward(X, W, b, None, want, M, N, K)
    every_other, wide = torch.zeros(2 * M, K, device=DEV, dtype=torch.bfloat16), torch.zeros(2, 3, K + 8, device=DEV, dtype=torch.bfloat16)
    every_other[::2], wide[..., :K] = X, X.view(2, 3, K)
    for x, ldx in ((X.reshape(-1), 0), (X.view(2, 3, K), 0), (every_other, 2 * K), (every_other[::2], 2 * K), (wide[..., :K], K + 8), (X.view(torch.int16), 0), (X.data_ptr(), 0)):
        got.zero_()
        plan.forward(x, W, b, None, got, M, N, K, ldx=ldx)
        assert torch.equal(got, want)
    plan.close()


def test_a_plan_for_few_rows_is_small(ccn):
    """Up to 64 rows the weights are read as they lie and a sum over the rows is never split: such a plan holds neither a copy of W
    (64 MiB here) nor that product's partial sums (32 MiB), and serves both directions."""
    M, N, K = 16, 4096, 8192
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    plan = ccn.LinearPlan(M, N, K)
    taken = free - torch.cuda.mem_get_info()[0]
    assert taken < 24 << 20, taken
    forward_case(ccn, M, N, K, "gelu", False, pad=3, shift=1, plan=plan)
    plan.close()
    backward_case(ccn, 64, 1000, 1504, "silu", False, pad=3, shift=1)
