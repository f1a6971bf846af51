"""The dense layer, its gradients and AdamW together, as a training program uses them: a block of two layers (gelu, then back to the
residual stream), 16-bit weight copies written by the optimizer and read by the next forward pass, gradients in 16 bits for one
layer and summed over two micro-batches in fp32 for the other.

The restatement follows the same roundings to bf16 in float64.  What is left between the two sides: fp32 sums (2^-24 per term) and
a bf16 value that such a difference pushes over a rounding border, one step of 2^-8 on rare elements of the pre-activations, dz
and the 16-bit gradients.  Gradients are compared at 2^-7 of their tensor's rms plus 2^-7 relative (two such steps; sums of 386 or more
terms average the rest).  The weights: with eps = 1 the update lr*m/(sqrt(v) + eps) moves by at most lr * 2 * |dg| when a gradient
moves by |dg|, per step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOKENS, H, F = 193, 136, 520        # per micro-batch; two of them
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.95, 1.0, 0.1


def bf(x):
    return x.to(torch.bfloat16).to(torch.float64)


class Block:
    def __init__(self, ccn, bits):
        g = torch.Generator(device=DEV)
        g.manual_seed(3)
        self.ccn, self.bits = ccn, bits
        self.w = [torch.randn(H, F, device=DEV, generator=g) * 0.1, torch.randn(F, device=DEV, generator=g) * 0.1,
                  torch.randn(F, H, device=DEV, generator=g) * 0.1, torch.randn(H, device=DEV, generator=g) * 0.1]
        self.w16 = [x.bfloat16() for x in self.w]
        self.lin = ccn.LinearPlan(TOKENS, max(H, F), max(H, F))
        counts = [x.numel() for x in self.w]
        # the first layer's weight gradient is 16-bit, so it and the rest are two steps of two plans
        self.plans = [ccn.AdamWPlan(counts[:1], bits=bits), ccn.AdamWPlan(counts[1:], decay=[0.0, 1.0, 0.0], bits=bits)]
        dt = torch.float32 if bits == 32 else torch.uint8
        self.state = [(torch.zeros(p.elems, device=DEV, dtype=dt), torch.zeros(p.elems, device=DEV, dtype=dt),
                       None if bits == 32 else torch.zeros(2 * p.blocks, device=DEV)) for p in self.plans]

    def passes(self, X, G, stream=None):
        """Forward and backward over the micro-batches: outputs and the gradients of the four tensors."""
        M = X.shape[1]
        e = lambda *s: torch.empty(*s, device=DEV, dtype=torch.bfloat16)  # noqa: E731
        db1, dW2, db2 = torch.zeros(F, device=DEV), torch.zeros(F, H, device=DEV), torch.zeros(H, device=DEV)
        dW1 = [e(H, F) for _ in range(2)]
        Y, dX = [], []
        for k in range(2):
            pre, h, y = e(M, F), e(M, F), e(M, H)
            self.lin.forward(X[k], self.w16[0], self.w[1], None, h, M, F, H, act="gelu", pre=pre, stream=stream)
            self.lin.forward(h, self.w16[2], self.w[3], X[k], y, M, H, F, stream=stream)
            dh, dx, db = e(M, F), e(M, H), torch.empty(F, device=DEV)
            self.lin.backward(G[k], None, h, self.w16[2], dh, dW2, db2, M, H, F, dw_f32=True, accumulate=True, stream=stream)
            self.lin.backward(dh, pre, X[k], self.w16[0], dx, dW1[k], db, M, F, H, act="gelu", stream=stream)
            db1 += db
            Y.append(y)
            dX.append(dx)
        return Y, dX, (dW1, db1, dW2, db2)

    def update(self, grads, t, stream=None):
        dW1, db1, dW2, db2 = grads
        for p, (m, v, s), g, g_type, w, w16 in ((self.plans[0], self.state[0], [[x] for x in dW1], "bf16", self.w[:1], self.w16[:1]),
                                                (self.plans[1], self.state[1], [[db1, dW2, db2]], "f32", self.w[1:], self.w16[1:])):
            p.step(p.tables(g, w, w16), m, v, LR, B1, B2, EPS, WD, t, scales=s, g_type=g_type, stream=stream)


def reference(X, G, w16, b1, b2):
    """float64 with bf16 roundings where the library rounds."""
    W1, W2 = w16[0].double(), w16[2].double()
    out = []
    dW2, db1, db2 = 0, 0, 0
    dW1 = []
    for k in range(2):
        x, g = X[k].double(), G[k].double()
        z = x @ W1 + b1.double()
        pre, h = bf(z), bf(z * torch.special.ndtr(z))
        y = h @ W2 + b2.double() + x
        dh = bf(g @ W2.t())
        slope = torch.special.ndtr(pre) + pre * torch.exp(-pre * pre / 2) / math.sqrt(2 * math.pi)
        dzf = dh * slope
        dz = bf(dzf)
        dW2, db2, db1 = dW2 + h.t() @ g, db2 + g.sum(0), db1 + dzf.sum(0)
        dW1.append(x.t() @ dz)
        out.append((y, dz @ W1.t()))
    return out, (dW1, db1, dW2, db2)


def close(got, want, what):
    got = got.double()
    tol = 2.0 ** -7 * (want.square().mean().sqrt() + want.abs())
    assert ((got - want).abs() <= tol).all(), (what, ((got - want).abs() / tol).max().item())


def data(g):
    return (torch.randn(2, TOKENS, H, device=DEV, generator=g).bfloat16(), (torch.randn(2, TOKENS, H, device=DEV, generator=g) * 0.05).bfloat16())


def test_three_steps(ccn):
    g = torch.Generator(device=DEV)
    g.manual_seed(9)
    blk = Block(ccn, 32)
    m = [torch.zeros_like(x, dtype=torch.float64) for x in blk.w]
    v = [torch.zeros_like(x, dtype=torch.float64) for x in blk.w]
    decay = [1.0, 0.0, 1.0, 0.0]
    for t in (1, 2, 3):
        X, G = data(g)
        before = [x.double().clone() for x in blk.w]
        out, want = reference(X, G, blk.w16, blk.w[1], blk.w[3])
        Y, dX, grads = blk.passes(X, G)
        torch.cuda.synchronize()
        for k in range(2):
            close(Y[k], out[k][0], "Y")
            close(dX[k], out[k][1], "dX")
            close(grads[0][k], want[0][k], "dW1")
        for name, a, b in zip(("db1", "dW2", "db2"), grads[1:], want[1:]):
            close(a, b, name)
        blk.update(grads, t)
        torch.cuda.synchronize()
        for i, gr in enumerate([grads[0][0].double() + grads[0][1].double()] + [x.double() for x in grads[1:]]):
            m[i] = B1 * m[i] + (1 - B1) * gr
            v[i] = B2 * v[i] + (1 - B2) * gr * gr
            w = before[i] * (1 - LR * WD * decay[i]) - LR * (m[i] / (1 - B1 ** t)) / ((v[i] / (1 - B2 ** t)).sqrt() + EPS)
            assert ((blk.w[i].double() - w).abs() <= 2.0 ** -20 * (before[i].abs() + LR * (1 + gr.abs()))).all(), ("w", i, t)
            assert torch.equal(blk.w16[i], blk.w[i].bfloat16())


def test_the_first_step_does_not_depend_on_the_moments_width(ccn):
    """From zero moments the update uses the step's own m and v before they are rounded: the same bits with 8 and with 32."""
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    X, G = data(g)
    a, b = Block(ccn, 32), Block(ccn, 8)
    for blk in (a, b):
        blk.update(blk.passes(X, G)[2], 1)
    torch.cuda.synchronize()
    for x, y in zip(a.w + a.w16, b.w + b.w16):
        assert torch.equal(x, y)
    X, G = data(g)
    for t in (2, 3):
        b.update(b.passes(X, G)[2], t)
    torch.cuda.synchronize()
    assert all(torch.isfinite(x).all() for x in b.w)


def test_a_recorded_step(ccn):
    """Both passes of both micro-batches and the update recorded once and replayed on new data, against the same calls made one by
    one (the library's calls alone are recorded: the sum of the two db is made by a kernel of torch's on the same stream, so the
    recording here is of one layer and its update)."""
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    M = TOKENS
    blocks = [Block(ccn, 8) for _ in range(2)]
    X, G = data(g)
    X, G = X[0], (torch.randn(M, F, device=DEV, generator=g) * 0.05).bfloat16()
    bufs = []
    for blk in blocks:
        e = lambda *s: torch.empty(*s, device=DEV, dtype=torch.bfloat16)  # noqa: E731
        bufs.append(dict(pre=e(M, F), h=e(M, F), dx=e(M, H), dW=e(H, F), db=torch.empty(F, device=DEV)))
    plans = [(ccn.AdamWPlan([H * F], bits=8), torch.zeros(-(-H * F // 256) * 256, device=DEV, dtype=torch.uint8), torch.zeros(-(-H * F // 256) * 256, device=DEV, dtype=torch.uint8),
              torch.zeros(2 * -(-H * F // 256), device=DEV)) for _ in blocks]
    tables = [p[0].tables([[b["dW"]]], blk.w[:1], blk.w16[:1]) for p, b, blk in zip(plans, bufs, blocks)]

    def calls(i, stream=None):
        blk, b, (p, m, v, s) = blocks[i], bufs[i], plans[i]
        blk.lin.forward(X, blk.w16[0], blk.w[1], None, b["h"], M, F, H, act="silu", pre=b["pre"], stream=stream)
        blk.lin.backward(G, b["pre"], X, blk.w16[0], b["dx"], b["dW"], b["db"], M, F, H, act="silu", stream=stream)
        p.step(tables[i], m, v, LR, B1, B2, 1e-8, WD, 1, scales=s, g_type="bf16", stream=stream)

    for i in range(2):
        calls(i)
    torch.cuda.synchronize()
    st = ccn.Stream()
    graph = ccn.Graph(st)
    with graph:
        calls(0, st.h)
    for rep in range(3):
        X.normal_(generator=g)
        G.normal_(generator=g)
        torch.cuda.synchronize()
        graph.launch()
        st.sync()
        calls(1)
        torch.cuda.synchronize()
        for k in bufs[0]:
            assert torch.equal(bufs[0][k], bufs[1][k]), (rep, k)
        assert torch.equal(blocks[0].w[0], blocks[1].w[0]) and torch.equal(plans[0][1], plans[1][1]) and torch.equal(plans[0][3], plans[1][3]), rep
    graph.close()
    st.close()


def test_two_plans_at_once_on_two_streams(ccn):
    """Calls on plans of their own do not disturb each other: the same calls one after the other give the same bits.  Rows that take
    the split sums, the joined few-row kernel and the pair kernel; AdamW steps with and without a flag launch."""
    g = torch.Generator(device=DEV)
    g.manual_seed(9)

    def layer(M, N, K):
        rand = lambda *sh: torch.randn(*sh, device=DEV, generator=g).bfloat16()  # noqa: E731
        x, w, dy = rand(M, K), rand(K, N), rand(M, N)
        plan = ccn.LinearPlan(M, N, K)

        def run(out, stream):
            for _ in range(8):
                plan.forward(x, w, None, None, out[0], M, N, K, act="silu", pre=out[1], stream=stream)
                plan.backward(dy, out[1], x, w, out[2], out[3], out[4], M, N, K, act="silu", stream=stream)

        def new():
            return [torch.zeros_like(dy), torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w), torch.zeros(N, device=DEV)]
        return plan, run, new

    def step(n, bits):
        grad, w0 = torch.randn(n, device=DEV, generator=g), torch.randn(n, device=DEV, generator=g)
        grad[n // 3] = math.inf
        plan = ccn.AdamWPlan([n], bits=bits)

        def run(out, stream):
            for t in range(1, 5):
                plan.step(plan.tables([[grad]], [out[0]]), out[1], out[2], LR, B1, B2, 1e-8, WD, t, scales=out[3] if bits == 8 else None,
                          overflow_flag=out[4], stream=stream)

        def new():
            m = torch.zeros(plan.elems, device=DEV, dtype=torch.uint8 if bits == 8 else torch.float32)
            return [w0.clone(), m, torch.zeros_like(m), torch.zeros(2 * plan.blocks, device=DEV), torch.zeros(1, device=DEV, dtype=torch.int32)]
        return plan, run, new

    jobs = [layer(16, 512, 4096), layer(48, 520, 2048), layer(300, 1500, 72), layer(2000, 136, 264), layer(7, 1000, 3000), step(100_000, 8), step(100_000, 32),
            step(3_000_000, 8)]
    for i in range(len(jobs)):
        (pa, ra, na), (pb, rb, nb) = jobs[i], jobs[(i + 1) % len(jobs)]
        alone_a, alone_b, a, b = na(), nb(), na(), nb()
        torch.cuda.synchronize()
        ra(alone_a, None)
        torch.cuda.synchronize()
        rb(alone_b, None)
        torch.cuda.synchronize()
        sa, sb = ccn.Stream(), ccn.Stream()
        ra(a, sa.h)
        rb(b, sb.h)
        torch.cuda.synchronize()
        for got, want in zip(a + b, alone_a + alone_b):
            assert torch.equal(got, want), i
        sa.close()
        sb.close()
    for plan, _run, _new in jobs:
        plan.close()
