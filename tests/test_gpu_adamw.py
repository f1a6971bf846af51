"""AdamW over many tensors (ccn_adamw_*), moments in fp32 and in 8 bits, against a float64 restatement.

Tolerances count fp32 roundings (2^-24 each): a gradient that is the sum of P buffers is off by (P+1) of them relative to
the sum of magnitudes; m and v by a few more; the update by those of m plus a dozen in the square root and division.  An
8-bit moment has to be within half a step (2^-4 relative, 2^-10 among the subnormals, in units of the scale) of the exact
value, plus what fp32 moved it by."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.98, eps=1e-8, wd=0.1)
MARK = 9.0


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def e4m3(codes):
    """All 256 OCP e4m3 codes, decoded by hand."""
    c = codes.long()
    s, e, m = c >> 7, (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1 + m / 8) * torch.pow(2.0, (e - 7).double()), m / 8 * 2.0 ** -6)
    return torch.where(s == 1, -v, v)


class Case:
    def __init__(self, ccn, counts, ranks, g_type="f32", copy=None, bits=32, decay=None, shift=0, seed=0, steps=0):
        self.ccn, self.counts, self.ranks, self.bits, self.g_type, self.copy = ccn, counts, ranks, bits, g_type, copy
        self.gen = gen(seed)
        self.plan = ccn.AdamWPlan(counts, decay=decay, bits=bits)
        assert self.plan.blocks == sum(-(-c // 256) for c in counts) and self.plan.elems == 256 * self.plan.blocks
        self.decay = decay or [1.0] * len(counts)
        n = self.plan.elems

        def buffers(dtype):
            """One buffer per tensor, `shift` elements into an allocation that is marked around it."""
            whole = [torch.full((shift + c + 8,), MARK, device=DEV, dtype=dtype) for c in counts]
            return whole, [x[shift:shift + c] for x, c in zip(whole, counts)]

        self.whole = []
        self.g = []
        for _ in range(ranks):
            whole, views = buffers(DT[g_type])
            self.g.append(views)
        whole, self.w = buffers(torch.float32)
        self.whole.append((whole, self.w))
        self.w16 = None
        if copy:
            whole, self.w16 = buffers(DT[copy])
            self.whole.append((whole, self.w16))
        for x in self.w:
            x.normal_(generator=self.gen)
        self.m = torch.zeros(n, device=DEV, dtype=torch.float32 if bits == 32 else torch.uint8)
        self.v = torch.zeros_like(self.m)
        self.scales = torch.zeros(2 * self.plan.blocks, device=DEV) if bits == 8 else None
        self.flag = torch.full((1,), 77, device=DEV, dtype=torch.int32)
        self.starts = []
        at = 0
        for c in counts:
            self.starts.append(at)
            at += -(-c // 256) * 256

    def new_gradients(self, scale=1.0):
        for r in self.g:
            for i, x in enumerate(r):
                x.copy_(torch.randn(x.shape, device=DEV, generator=self.gen) * (scale * 10.0 ** (i % 3 - 1)))

    def state(self):
        """w, m, sqrt(v) per tensor, float64."""
        if self.bits == 32:
            m, r = self.m.double(), self.v.double().sqrt()
        else:
            b = self.plan.blocks
            s = self.scales.double().view(2, b, 1)
            m, r = (e4m3(self.m).view(b, 256) * s[0]).view(-1), (e4m3(self.v).view(b, 256) * s[1]).view(-1)
        cut = lambda x: [x[o:o + c] for o, c in zip(self.starts, self.counts)]  # noqa: E731
        return [x.double().clone() for x in self.w], cut(m), cut(r)

    def step(self, t, inv_scale=1.0, grad_scale=None, stream=None, flag=True, **hyper):
        h = {**HYPER, **hyper}
        self.plan.step(self.plan.tables(self.g, self.w, self.w16), self.m, self.v, h["lr"], h["beta1"], h["beta2"], h["eps"], h["wd"], t, scales=self.scales,
                       g_type=self.g_type, w16_type=self.copy or "bf16", inv_scale=inv_scale, grad_scale=grad_scale, overflow_flag=self.flag if flag else None,
                       stream=stream)

    def check(self, before, t, scale=1.0, bad=None, **hyper):
        """The state against the step from `before` with the present gradients.  bad: per tensor, elements left out."""
        h = {**HYPER, **hyper}
        torch.cuda.synchronize()
        w0s, m0s, r0s = before
        w1s, m1s, r1s = self.state()
        P, b1, b2 = self.ranks, h["beta1"], h["beta2"]
        for i, c in enumerate(self.counts):
            if c == 0:
                continue
            g = sum(r[i].double() for r in self.g) * scale
            ga = sum(r[i].double().abs() for r in self.g) * scale
            w0, m0, v0 = w0s[i], m0s[i], r0s[i].square()
            m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
            mh, vh = m / (1 - b1 ** t), v / (1 - b2 ** t)
            den = vh.sqrt() + h["eps"]
            w = w0 * (1 - h["lr"] * h["wd"] * self.decay[i]) - h["lr"] * mh / den
            if bad is not None:
                w, m, v = (torch.where(bad[i], o, x) for o, x in ((w0, w), (m0, m), (v0, v)))
            em = (P + 6) * U * (b1 * m0.abs() + (1 - b1) * ga) + 1e-44
            ev = (2 * P + 10) * U * (b2 * v0 + (1 - b2) * ga * ga) + 1e-44
            r = v.sqrt()
            er = torch.where(r > 0, ev / r.clamp_min(1e-300), torch.zeros_like(r)) + 2 * U * r
            eu = em / (1 - b1 ** t) / den + (mh / den).abs() * (er / r.clamp_min(1e-300) + 16 * U)
            ew = 4 * U * w0.abs() + 2 * U * w.abs() + h["lr"] * eu + 1e-44
            if bad is not None:
                fine = ~bad[i]
            else:
                fine = torch.ones_like(w, dtype=torch.bool)
            assert torch.isfinite(w1s[i]).all()
            assert ((w1s[i] - w).abs() <= ew)[fine].all(), ("w", i, ((w1s[i] - w).abs() / ew)[fine].max().item())
            assert torch.equal(w1s[i][~fine], w0[~fine])
            if self.copy:
                assert torch.equal(self.w16[i], self.w[i].to(DT[self.copy])), ("w16", i)
            if self.bits == 32:
                assert ((m1s[i] - m).abs() <= em).all(), ("m", i)
                assert ((r1s[i] - r).abs() <= er).all(), ("v", i)
                continue
            nb = -(-c // 256)
            o = self.starts[i] // 256
            for name, got, x, ex, sc in (("m", self.m, m, em, self.scales[o:o + nb]), ("v", self.v, r, er, self.scales[self.plan.blocks + o:self.plan.blocks + o + nb])):
                pad = torch.zeros(nb * 256, device=DEV, dtype=torch.float64)
                xp, ep = pad.clone(), pad.clone()
                xp[:c], ep[:c] = x, ex
                xp, ep = xp.view(nb, 256), ep.view(nb, 256)
                top = xp.abs().amax(1)
                assert ((sc.double() - top / 448).abs() <= 2 * U * top / 448 + ep.amax(1) / 448 + 1e-44).all(), (name, i, "scale")
                s = sc.double()[:, None].clamp_min(1e-300)
                y, val = xp / s, e4m3(got[self.starts[i]:self.starts[i] + nb * 256]).view(nb, 256)
                step = torch.maximum(torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3), torch.tensor(2.0 ** -9, device=DEV, dtype=torch.float64))
                tol = step / 2 + ep / s + 8 * U * y.abs()
                if name == "v":   # not zero: at least the smallest code
                    tol = torch.where(xp > 0, torch.maximum(tol, 2.0 ** -9 - y + tol), tol)
                live = s > 1e-300
                assert (((val - y).abs() <= tol) | ~live).all(), (name, i, ((val - y).abs() / tol).max().item())
                if name == "v":
                    assert ((val > 0) == (xp > 0)).all() or (ep > xp)[(val > 0) != (xp > 0)].all(), (name, i, "zero")
                assert not val.view(-1)[c:].any()

    def nothing_else_written(self):
        for whole, views in self.whole:
            for buf, v in zip(whole, views):
                keep = v.clone()
                v.fill_(MARK)
                assert bool((buf == MARK).all())
                v.copy_(keep)


COUNTS = [1, 255, 256, 257, 0, 511, 512, 513, 1000, 70001, 3]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ranks", [1, 2, 3, 5, 9, 16])
def test_ranks_and_types(ccn, bits, ranks):
    for j, (g_type, copy) in enumerate((("f32", None), ("bf16", "bf16"), ("f16", "f16"))):
        c = Case(ccn, COUNTS, ranks, g_type, copy, bits, decay=[float(k % 2) for k in range(len(COUNTS))], seed=ranks + j)
        for t in (1, 2, 3):
            c.new_gradients()
            before = c.state()
            c.step(t, inv_scale=0.25)
            c.check(before, t, scale=0.25)
            assert c.flag.item() == 0
        c.nothing_else_written()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [1, 2, 3, 4, 8])
def test_alignments(ccn, bits, shift):
    for g_type, copy in (("f32", "bf16"), ("bf16", None), ("f16", "f16")):
        c = Case(ccn, COUNTS, 2, g_type, copy, bits, shift=shift, seed=shift)
        c.new_gradients()
        before = c.state()
        c.step(4)
        c.check(before, 4)
        c.nothing_else_written()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(ccn, bits):
    """More tensors than a wavefront looks at, one tile each, among longer ones."""
    counts = [(i * 37) % 300 for i in range(700)] + [100_000] + [5] * 130
    c = Case(ccn, counts, 1, "bf16", "bf16", bits)
    for t in (1, 2):
        c.new_gradients()
        before = c.state()
        c.step(t)
        c.check(before, t)
    c.nothing_else_written()


@pytest.mark.parametrize("bits", [32, 8])
def test_large_tensor(ccn, bits):
    c = Case(ccn, [(1 << 24) + 77, 1 << 20], 1, "bf16", "bf16", bits)
    for t in (1, 2):
        c.new_gradients(1e-3)
        before = c.state()
        c.step(t)
        c.check(before, t)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(ccn, bits):
    for g_type in ("f32", "bf16", "f16"):
        c = Case(ccn, [1000, 300], 2, g_type, "f16" if g_type == "f16" else "bf16", bits)
        c.new_gradients()
        c.step(1)
        c.new_gradients()
        bad = [torch.zeros(n, dtype=torch.bool, device=DEV) for n in c.counts]
        for i, e, r, x in ((0, 0, 0, math.inf), (0, 255, 1, -math.inf), (0, 999, 0, math.nan), (1, 7, 1, math.nan)):
            c.g[r][i][e] = x
            bad[i][e] = True
        if g_type != "f16":     # finite, but its square is not
            c.g[0][1][100], c.g[1][1][100] = 2.0 ** 100, 0.0
            bad[1][100] = True
        before = c.state()
        old = [x.clone() for x in c.w]
        c.step(2)
        torch.cuda.synchronize()
        assert c.flag.item() == 1
        for r in c.g:
            for i in range(2):
                r[i][bad[i]] = 0      # the restatement leaves them out
        c.check(before, 2, bad=bad)
        for i in range(2):
            assert torch.equal(c.w[i][bad[i]], old[i][bad[i]])
        c.step(3)
        torch.cuda.synchronize()
        assert c.flag.item() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_grad_scale_on_the_device(ccn, bits):
    c = Case(ccn, [777, 4096], 1, "f32", None, bits)
    s = torch.tensor([0.125], device=DEV)
    for t in (1, 2):
        c.new_gradients()
        before = c.state()
        c.step(t, inv_scale=0.5, grad_scale=s, flag=False)
        c.check(before, t, scale=0.0625)


def test_zero_gradients_zero_state(ccn):
    """0 / (0 + eps): nothing moves but by the decay; with no eps and no gradient the update would be 0/0 and the formula says NaN,
    so eps > 0 is what is tested."""
    for bits in (32, 8):
        c = Case(ccn, [300], 1, bits=bits)
        c.g[0][0].zero_()
        w0 = c.w[0].clone()
        c.step(1, wd=0.0)
        torch.cuda.synchronize()
        assert torch.equal(c.w[0], w0) and not c.m.any() and not c.v.any() and c.flag.item() == 0


def test_small_values_do_not_vanish(ccn):
    """8 bits: an element 10^6 smaller than its block's largest keeps a second moment that is not zero, so that its update stays
    bounded by the first moment it has."""
    c = Case(ccn, [256], 1, bits=8)
    for t in range(1, 30):
        c.g[0][0].fill_(1e-7)
        c.g[0][0][3] = 1.0
        w0 = c.w[0].clone()
        c.step(t, wd=0.0)
        torch.cuda.synchronize()
        assert (c.w[0] - w0).abs().max() <= 4e-3, t     # |update| <= lr * a few


def test_follows_the_32_bit_trajectory(ccn):
    """Both widths on a quadratic from the same start end near its minimum."""
    target = torch.randn(5000, device=DEV, generator=gen(5))
    for bits in (32, 8):
        c = Case(ccn, [5000], 1, bits=bits)
        for t in range(1, 201):
            c.g[0][0].copy_(c.w[0] - target)
            c.step(t, lr=5e-2, wd=0.0, flag=False)
        assert (c.w[0] - target).abs().mean() < 0.05


def test_e4m3_codes(ccn):
    """Every code through a step that changes nothing (beta 0 would, so: no gradient weight): decode and encode agree with the
    definition for all 256 values, block by block."""
    c = Case(ccn, [256 * 2], 1, bits=8)
    codes = torch.arange(256, device=DEV, dtype=torch.uint8)
    codes[(codes & 0x7f) == 0x7f] = 0x7e       # the two NaN codes are no state
    roots = (codes & 0x7f)
    c.m[:256], c.v[:256] = codes, roots
    c.m[256:], c.v[256:] = codes.flip(0), roots.flip(0)
    c.scales.copy_(torch.tensor([1.0, 2.0 ** -10, 2.0 ** -8, 2.0 ** -20], device=DEV))
    c.g[0][0].zero_()
    c.step(1, beta1=0.5, beta2=0.25, lr=0.0, wd=0.0)
    torch.cuda.synchronize()
    # m halves: the scale does, the codes stay; sqrt(v) halves too
    assert torch.equal(c.m[:256] & 0x7f, codes & 0x7f) and torch.equal(e4m3(c.m[:256]), e4m3(codes))
    assert torch.equal(c.v[:256], roots) and torch.equal(c.v[256:], roots.flip(0))
    assert torch.allclose(c.scales, torch.tensor([0.5, 2.0 ** -11, 2.0 ** -9, 2.0 ** -21], device=DEV), rtol=2.0 ** -22)


def test_streams_and_recording(ccn):
    """A recorded step replays on the buffers it was made with; other pointers are refused while recording and afterwards."""
    for bits in (32, 8):
        st = ccn.Stream()
        a, b = (Case(ccn, [1000, 70001], 2, "bf16", "bf16", bits, seed=3) for _ in range(2))
        for c in (a, b):
            c.new_gradients()
        torch.cuda.synchronize()
        graph = ccn.Graph(st)
        with pytest.raises(ccn.CoconetError):
            with graph:
                a.step(1, stream=st.h)           # the plan has not seen these pointers
        a.step(1)
        b.step(1)
        torch.cuda.synchronize()
        graph = ccn.Graph(st)
        with graph:
            a.step(2, stream=st.h)
        for rep in range(3):
            for x, y in zip((x for r in a.g for x in r), (y for r in b.g for y in r)):
                x.normal_(generator=a.gen)
                y.copy_(x)
            torch.cuda.synchronize()
            graph.launch()
            st.sync()
            b.step(2)
            torch.cuda.synchronize()
            for x, y in zip(a.w + a.w16 + [a.m, a.v, a.flag], b.w + b.w16 + [b.m, b.v, b.flag]):
                assert torch.equal(x, y), rep
        a.w = [x.clone() for x in a.w]
        with pytest.raises(ccn.CoconetError) as e:
            a.step(3)
        assert e.value.code == ccn.CCN_EINVAL
        graph.close()
        st.close()


def test_pointers_may_change_between_steps(ccn):
    c = Case(ccn, [5000, 123], 1, "bf16", None, 8)
    for t in range(1, 8):
        c.g = [[torch.randn(n, device=DEV, generator=c.gen).bfloat16() for n in c.counts]]
        before = c.state()
        c.step(t)
        c.check(before, t)


def test_refusals(ccn):
    c = Case(ccn, [300, 0, 40], 2, "bf16", "bf16", 8)
    c.new_gradients()
    old = [x.clone() for x in c.w]
    E = ccn.CCN_EINVAL
    gt, P, wt, ht = c.plan.tables(c.g, c.w, c.w16)

    def refused(**k):
        a = dict(tables=(gt, P, wt, ht), m=c.m, v=c.v, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, wd=0.0, step=1, scales=c.scales, g_type="bf16")
        a.update(k)
        with pytest.raises(ccn.CoconetError) as e:
            c.plan.step(**a)
        assert e.value.code == E, k

    refused(tables=(gt, 0, wt, ht))
    refused(tables=(gt, 17, wt, ht))
    refused(step=0)
    refused(m=None)
    refused(v=c.v.data_ptr() + 1)
    refused(scales=None)
    refused(beta1=1.0)
    refused(beta2=-0.1)
    refused(eps=-1.0)
    refused(w16_type="f32")
    refused(tables=c.plan.tables([[x.data_ptr() + 1 for x in r] for r in c.g], c.w, c.w16))
    refused(tables=c.plan.tables(c.g, [0, c.w[1], c.w[2]], c.w16))
    refused(tables=c.plan.tables(c.g, [x.data_ptr() + 2 for x in c.w], c.w16))
    refused(grad_scale=c.scales.data_ptr() + 1)
    refused(overflow_flag=c.flag.data_ptr() + 1)
    p32 = ccn.AdamWPlan([300, 0, 40])
    m32 = torch.zeros(p32.elems, device=DEV)
    with pytest.raises(ccn.CoconetError):
        p32.step((gt, P, wt, ht), m32, m32, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, scales=c.scales, g_type="bf16")   # scales of 32-bit moments
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(old, c.w)) and not c.m.any()
    empty = ccn.AdamWPlan([0, 0], bits=8)
    assert empty.elems == 0 and empty.blocks == 0
    empty.step(empty.tables([[None, None]], [None, None]), None, None, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, overflow_flag=c.flag)
    torch.cuda.synchronize()
    assert c.flag.item() == 0


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("blocks", [1, 31, 32, 33, 1024, 1055, 8191, 8192, 8193, 20000])
def test_flag_at_every_size(ccn, bits, blocks):
    """The flag is written by every call, whatever it held: 1 for a gradient that is not finite in any block, else 0."""
    n = 256 * blocks - 100
    plan = ccn.AdamWPlan([n], bits=bits)
    g = torch.randn(n, device=DEV, generator=gen(blocks))
    w, flag = torch.zeros(n, device=DEV), torch.full((2,), 55, device=DEV, dtype=torch.int32)
    m = torch.zeros(plan.elems, device=DEV, dtype=torch.uint8 if bits == 8 else torch.float32)
    v, scales = torch.zeros_like(m), torch.zeros(2 * blocks, device=DEV) if bits == 8 else None
    tables = plan.tables([[g]], [w])
    st = ccn.Stream()

    def step(stream=None):
        plan.step(tables, m, v, 1e-3, 0.9, 0.98, 1e-8, 0.1, 1, scales=scales, overflow_flag=flag, stream=stream)

    step()
    torch.cuda.synchronize()
    with ccn.Graph(st) as graph:
        step(st.h)
    for at in (None, 0, n - 1, None, n // 2, (n * 5) // 7, None):
        for run in (step, graph.launch):
            old = g[at].clone() if at is not None else None
            if at is not None:
                g[at] = math.inf if at else math.nan
            flag[0] = 7 if at is None else 0
            torch.cuda.synchronize()
            run()
            st.sync()
            torch.cuda.synchronize()
            assert flag.tolist() == [0 if at is None else 1, 55], at
            if at is not None:
                g[at] = old
    g[0], g[n - 1] = -math.inf, 1e38     # two at once, the square of the second alone is not finite
    torch.cuda.synchronize()
    step()
    torch.cuda.synchronize()
    assert flag[0].item() == 1
    graph.close()
    plan.close()
    st.close()


@pytest.mark.parametrize("bits", [8, 32])
def test_offsets_past_32_bits(ccn, bits):
    """More blocks than a row of the grid takes (2^33 elements; 2^24 with fp32 moments: 2^32): tensors with the same
    values end alike, whichever their place."""
    each, n = (1 << 30, 8) if bits == 8 else (1 << 29, 8)
    counts = [each] * n + [1000]
    need = sum(counts) * (4 + (2 if bits == 8 else 8)) + 2 * each
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip("not enough memory free")
    g = torch.randn(each, device=DEV, generator=gen(3)).bfloat16()
    first = torch.randn(each, device=DEV, generator=gen(4))
    w = [first.clone() for _ in range(n)] + [first[:1000].clone()]
    plan = ccn.AdamWPlan(counts, bits=bits)
    m = torch.zeros(plan.elems, device=DEV, dtype=torch.uint8 if bits == 8 else torch.float32)
    v = torch.zeros_like(m)
    scales = torch.zeros(2 * plan.blocks, device=DEV) if bits == 8 else None
    h = HYPER
    plan.step(plan.tables([[g] * n + [g[:1000]]], w), m, v, h["lr"], h["beta1"], h["beta2"], h["eps"], h["wd"], 1, scales=scales, g_type="bf16")
    torch.cuda.synchronize()
    assert not torch.equal(w[0], first)
    for i in range(1, n):
        assert torch.equal(w[i], w[0]), i
        assert torch.equal(m[i * each:(i + 1) * each], m[:each]) and torch.equal(v[i * each:(i + 1) * each], v[:each]), i
    assert torch.equal(w[n], w[0][:1000]) and torch.equal(m[n * each:][:512], m[:512])
    plan.close()
    # the first tensor alone, as the other tests check it
    plan = ccn.AdamWPlan([each], bits=bits)
    m1, v1 = torch.zeros_like(m[:each]), torch.zeros_like(m[:each])
    s1 = torch.zeros(2 * plan.blocks, device=DEV) if bits == 8 else None
    plan.step(plan.tables([[g]], [first]), m1, v1, h["lr"], h["beta1"], h["beta2"], h["eps"], h["wd"], 1, scales=s1, g_type="bf16")
    torch.cuda.synchronize()
    assert torch.equal(first, w[0]) and torch.equal(m1, m[:each]) and torch.equal(v1, v[:each])
    plan.close()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("last", [3, 8300 * 256 - 7], ids=["few-blocks", "many-blocks"])
def test_what_lies_behind_a_tensors_end(ccn, bits, last):
    """Moment arrays that hold anything behind the tensors' ends (a state restored into uninitialised memory): the flag and the
    live elements are those of a step over zeros there."""
    counts = [1, 255, 257, 1000, 513, 256, last]
    a, b = (Case(ccn, counts, 2, "bf16", "bf16", bits, seed=6) for _ in range(2))
    behind = torch.ones(a.plan.elems, dtype=torch.bool, device=DEV)
    for o, n in zip(a.starts, counts):
        behind[o:o + n] = False
    for t, fill in enumerate((None, math.nan, math.inf, -math.inf, 3e38), 1):
        for c in (a, b):
            c.gen = gen(t)
            c.new_gradients()
        if fill is not None:
            # 8 bits: the two NaN codes, and the largest values
            code = {math.nan: 0x7f, math.inf: 0xff, -math.inf: 0xfe}.get(fill, 0x7e)
            for x in (a.m, a.v):
                x[behind] = fill if bits == 32 else code
        for c in (a, b):
            c.step(t)
        torch.cuda.synchronize()
        assert a.flag.item() == 0 and b.flag.item() == 0, fill
        for x, y in zip(a.w + a.w16 + [a.m[~behind], a.v[~behind]], b.w + b.w16 + [b.m[~behind], b.v[~behind]]):
            assert torch.equal(x, y), fill
        if bits == 8:
            assert torch.equal(a.scales, b.scales) and not a.m[behind].any() and not a.v[behind].any(), fill


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("beta2", [0.0, 0.5, 0.98, 0.9999])
def test_the_flags_border(ccn, bits, beta2):
    """The square of a gradient overflows fp32 from 2^64 on, whatever beta2: such an element keeps its state and sets the flag, the
    float below does neither."""
    below = (2.0 - 2.0 ** -23) * 2.0 ** 63
    for x, bad in ((below, False), (-below, False), (2.0 ** 64, True), (3e19, True), (-5e20, True)):
        c = Case(ccn, [700, 20], 1, "f32", None, bits, seed=2)
        c.new_gradients()
        c.step(1, beta2=beta2)
        c.new_gradients()
        c.g[0][0][300] = x
        old, before = [w.clone() for w in c.w], c.state()
        c.step(2, beta2=beta2)
        torch.cuda.synchronize()
        assert c.flag.item() == int(bad), (x, beta2)
        assert (c.w[0][300] == old[0][300]).item() == bad and not torch.equal(c.w[1], old[1])
        now = c.state()
        if bad and bits == 32:
            assert now[1][0][300] == before[1][0][300] and now[2][0][300] == before[2][0][300]
        assert all(torch.isfinite(y).all() for part in now for y in part)


def test_a_second_moment_that_is_not_finite(ccn):
    """A restored v that is inf or NaN says nothing about the gradient: no flag, and the element stays as it is."""
    c = Case(ccn, [700], 1)
    c.new_gradients()
    c.step(1)
    c.v[5], c.v[400], c.v[699] = math.inf, math.nan, math.inf
    at = torch.tensor([5, 400, 699], device=DEV)
    w, m = c.w[0].clone(), c.m.clone()
    c.new_gradients()
    c.step(2)
    torch.cuda.synchronize()
    assert c.flag.item() == 0
    assert torch.equal(c.w[0][at], w[at]) and torch.equal(c.m[at], m[at]) and not torch.isfinite(c.v[at]).any()
    fine = torch.ones(700, dtype=torch.bool, device=DEV)
    fine[at] = False
    assert torch.isfinite(c.w[0]).all() and not torch.equal(c.w[0][fine], w[fine])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("rate", [1e-7, 4.7e-8, 2e-8, 3.3e-4])
def test_decay_is_not_rounded(ccn, bits, rate):
    """A step without gradients: w*(1 - lr*wd), off by half a step of the result and by three roundings of the decay itself."""
    n, lr = 1 << 20, 1e-5
    c = Case(ccn, [n], 1, bits=bits)
    c.g[0][0].zero_()
    w0 = c.w[0].double()
    c.step(1, lr=lr, wd=rate / lr)
    torch.cuda.synchronize()
    want = w0 * (1 - rate)
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 25)
    d = (c.w[0].double() - want).abs()
    assert (d <= half + 3 * U * rate * w0.abs()).all(), (d / half).max().item()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("rate", [1e-7, 2e-8])
def test_decay_beside_updates(ccn, bits, rate):
    """Updates of all sizes (from a state of their own): what rounds the new weights, each to half a step of 2^-23, averages out over
    2^20 of them (6 sigma of a uniform error), so that the mean shows a decay far below a weight's last bit.  The update itself is off
    by some 64 roundings at most."""
    n, lr = 1 << 20, 1e-5
    c = Case(ccn, [n], 1, bits=bits)
    for t in (1, 2):
        c.new_gradients()
        c.step(t, lr=0.0, wd=0.0)
    c.w[0].copy_(1 + torch.rand(n, device=DEV, generator=c.gen) * 0.99)
    torch.cuda.synchronize()
    (w0,), (m0,), (r0,) = c.state()
    c.new_gradients()
    c.step(3, lr=lr, wd=rate / lr)
    torch.cuda.synchronize()
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    g = c.g[0][0].double()
    m, v = b1 * m0 + (1 - b1) * g, b2 * r0.square() + (1 - b2) * g * g
    u = lr * (m / (1 - b1 ** 3)) / ((v / (1 - b2 ** 3)).sqrt() + HYPER["eps"])
    d = c.w[0].double() - (w0 - rate * w0 - u)
    assert d.mean().abs() <= 6 * 2.0 ** -23 / math.sqrt(12 * n) + 64 * U * u.abs().mean() + 3 * U * rate * w0.mean(), d.mean().item()


def test_tensors_that_are_not_what_they_are_taken_for(ccn):
    """Types, orders and sizes of the Python call's tensors are refused; transposed tensors are taken where all of a tensor's arrays
    are, element for element as they lie."""
    c = Case(ccn, [300, 40], 1, "bf16", "bf16", 8)
    c.new_gradients()
    old = [x.clone() for x in c.w]

    def refused(code, f, *a, **k):
        with pytest.raises(ccn.CoconetError) as e:
            f(*a, **k)
        assert e.value.code == code

    E, R = ccn.CCN_EINVAL, ccn.CCN_ERANGE
    refused(E, c.plan.tables, [[x.float() for x in c.g[0][:1]] + c.g[0][1:]], c.w, c.w16)
    refused(E, c.plan.tables, c.g, [x.bfloat16() for x in c.w], c.w16)
    refused(E, c.plan.tables, [[x.cpu() for x in c.g[0]]], c.w, c.w16)
    refused(R, c.plan.tables, c.g, [c.w[0], c.w[1][:39]], c.w16)
    tables = c.plan.tables(c.g, c.w, c.w16)
    h = (1e-3, 0.9, 0.98, 1e-8, 0.1, 1)
    good = dict(scales=c.scales, g_type="bf16", w16_type="bf16")
    refused(E, c.plan.step, tables, c.m, c.v, *h, **{**good, "g_type": "f32"})
    refused(E, c.plan.step, tables, c.m, c.v, *h, **{**good, "w16_type": "f16"})
    refused(E, c.plan.step, tables, c.m.float(), c.v, *h, **good)
    refused(R, c.plan.step, tables, c.m, c.v[:-1], *h, **good)
    refused(R, c.plan.step, tables, c.m, c.v, *h, **{**good, "scales": c.scales[1:]})
    refused(E, c.plan.step, tables, c.m, c.v, *h, **good, grad_scale=torch.ones(1, device=DEV, dtype=torch.float64))
    refused(E, c.plan.step, tables, c.m, c.v, *h, **good, overflow_flag=torch.zeros(1, device=DEV))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(old, c.w)) and not c.m.any()

    plan, out = ccn.AdamWPlan([300]), []
    g, w = torch.randn(20, 15, device=DEV, generator=c.gen), torch.randn(20, 15, device=DEV, generator=c.gen)
    for turn in (lambda x: x, lambda x: x.t()):
        m, v, x = torch.zeros(plan.elems, device=DEV), torch.zeros(plan.elems, device=DEV), w.clone()
        plan.step(plan.tables([[turn(g)]], [turn(x)]), m, v, *h)
        out.append(x)
    assert torch.equal(*out) and not torch.equal(out[0], w)
    refused(E, plan.tables, [[g.t()]], [w])
    m, v, x = torch.zeros(plan.elems, device=DEV), torch.zeros(plan.elems, device=DEV), w.clone()
    plan.step(((ctypes.c_void_p * 1)(g.data_ptr()), 1, (ctypes.c_void_p * 1)(x.data_ptr()), None), m, v, *h)      # a caller's own tables
    assert torch.equal(x, out[0])
