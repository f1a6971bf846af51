"""Cases of the training and serving step of a dense layer, and how one pass of each is run.

The operators:
  linear     Y = act(X.W + bias) + resid, the pre-activation kept on request; one token to a whole batch of sequences
  backward   the same layer's gradients: dX, dW (16-bit, or added to an fp32 sum) and db, from dY and the kept pre-activation
  adamw      one AdamW step over many tensors at once, moments in fp32 or in 8 bits with a scale per 256 elements

`own` False runs them in elementary torch operations in fp32, True through the library.  X, W, dY are [rows x columns],
row-major, each inside rows of `pad` more elements.  W is [K x N].

The 8-bit moments: each tensor is cut into blocks of 256 elements (the last one of a tensor is filled up with zeros); a
block holds m / sm and sqrt(v) / sr as e4m3 values, sm = max|m| / 448 and sr = max sqrt(v) / 448, each rounded to nearest
even; a sqrt(v) that is not zero is never held as zero.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 256            # elements of one scale, and what every tensor's moments are padded to
E4M3_MAX = 448.0
E4M3_TINY = 2.0 ** -9  # its smallest value above zero
LARGEST = 8192 * 8192 * 4096   # rows x inner x columns of the largest product
LR, BETA1, BETA2, EPS, WD = 3e-4, 0.9, 0.95, 1e-8, 0.1


def listed():
    return [
        # one token through a layer of the 8-way split MLP whose rows are 8192 long (serving, latency)
        {"name": "linear-1-token", "op": "linear", "M": 1, "K": 1024, "N": 8192, "type": "bf16", "act": "gelu_tanh", "bias": True, "resid": False, "keep": False, "pad": 0},
        # a small batch of sequences, one token each, back down to the residual stream
        {"name": "linear-16-tokens", "op": "linear", "M": 16, "K": 8192, "N": 4096, "type": "f16", "act": "none", "bias": True, "resid": True, "keep": False, "pad": 0},
        # a ragged batch: sizes that no tile divides, rows that start anywhere
        {"name": "linear-ragged", "op": "linear", "M": 777, "K": 1537, "N": 2049, "type": "bf16", "act": "gelu", "bias": True, "resid": True, "keep": True, "pad": 0},
        # the forward pass of a training step: 8192 tokens, hidden size 8192, one rank's half of the inner size
        {"name": "linear-8192-tokens", "op": "linear", "M": 8192, "K": 8192, "N": 4096, "type": "bf16", "act": "gelu_tanh", "bias": True, "resid": False, "keep": True, "pad": 0},
        # gradients of a small layer (a probe, an adapter, a reward head's trunk)
        {"name": "backward-small", "op": "backward", "M": 256, "K": 1024, "N": 1024, "type": "f16", "act": "relu", "grad": "f16", "pad": 0},
        # gradients of the ragged layer
        {"name": "backward-ragged", "op": "backward", "M": 1001, "K": 515, "N": 2049, "type": "bf16", "act": "gelu", "grad": "bf16", "pad": 3},
        # the out-projection, which has no activation, with its weight gradients summed over micro-batches in fp32
        {"name": "backward-fp32-sum", "op": "backward", "M": 4096, "K": 4096, "N": 2048, "type": "bf16", "act": "none", "grad": "f32", "pad": 0},
        # the backward pass of the training step above
        {"name": "backward-8192-tokens", "op": "backward", "M": 8192, "K": 8192, "N": 4096, "type": "bf16", "act": "gelu_tanh", "grad": "bf16", "pad": 0},
        # a small model's tensors: biases and norms beside matrices, odd sizes, fp32 gradients of two ranks
        {"name": "adamw-small", "op": "adamw", "bits": 32, "tensors": 48, "total": 500_000, "mix": 7, "ranks": 2, "type": "f32", "copy": "none"},
        # half of the benchmark's 2^28 parameters in its buffers of 2^20, 16-bit gradients and a 16-bit copy of the weights
        {"name": "adamw-large", "op": "adamw", "bits": 32, "tensors": 128, "total": 1 << 27, "mix": 0, "ranks": 1, "type": "bf16", "copy": "bf16"},
        # the same with the moments in 8 bits: a middling model with fp16 gradients of two ranks, and the large one
        {"name": "adamw8-middle", "op": "adamw", "bits": 8, "tensors": 150, "total": 12_000_000, "mix": 5, "ranks": 2, "type": "f16", "copy": "f16"},
        {"name": "adamw8-large", "op": "adamw", "bits": 8, "tensors": 128, "total": 1 << 27, "mix": 0, "ranks": 1, "type": "bf16", "copy": "bf16"},
    ]


def _size(rng, low, high):
    """A size, spread over its logarithm: any number, a multiple of 8, or of 128."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    step = rng.choice((1, 1, 8, 128))
    return min(high, max(low, n // step * step if n >= step else n))


def draw(rng):
    op = rng.choice(("linear", "backward", "adamw", "adamw"))
    if op == "adamw":
        n = _size(rng, 1, 250)
        return {"op": op, "bits": rng.choice((8, 32)), "tensors": n, "total": max(4 * n, _size(rng, 5000, 1 << 26)), "mix": rng.randint(1, 10 ** 6),
                "ranks": rng.choice((1, 1, 2, 3)), "type": rng.choice(("bf16", "f16", "f32")), "copy": rng.choice(("none", "bf16", "f16"))}
    while True:
        M, K, N = _size(rng, 1, 8192), _size(rng, 64, 8192), _size(rng, 64, 8192)
        if M * K * N <= LARGEST:
            break
    case = {"op": op, "M": M, "K": K, "N": N, "type": rng.choice(("bf16", "bf16", "f16")),
            "act": rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")), "pad": rng.choice((0, 0, 8, 3))}
    if op == "linear":
        case.update(bias=rng.random() < 0.8, resid=rng.random() < 0.5, keep=rng.random() < 0.5)
    else:
        case["grad"] = "f32" if case["act"] == "none" else case["type"]
    return case


def _counts(case):
    """The tensors' element counts: equal ones (mix 0), or sizes spread over orders of magnitude."""
    n, total = case["tensors"], case["total"]
    if case["mix"] == 0:
        return [total // n] * n
    r = random.Random(case["mix"])
    share = [math.exp(r.gauss(0.0, 2.0)) for _ in range(n)]
    return [max(1, int(total * s / sum(share))) for s in share]


def _rows(gen, rows, cols, pad, scale, dtype):
    """A [rows x cols] matrix inside rows of cols + pad elements."""
    x = torch.empty(rows, cols + pad, device="cuda", dtype=torch.float32).normal_(0.0, scale, generator=gen)
    return x.to(dtype)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    if case["op"] == "adamw":
        counts = _counts(case)
        blocks = [-(-c // BLOCK) for c in counts]
        nb = sum(blocks)
        starts = [0]
        for b in blocks:
            starts.append(starts[-1] + b * BLOCK)
        inside = torch.zeros(nb * BLOCK, dtype=torch.bool, device="cuda")
        for o, c in zip(starts, counts):
            inside[o:o + c] = True
        # weights of 1-d tensors (every third one here) are not decayed; each tensor's gradients have a size of their own
        decay = [0.0 if i % 3 == 2 else 1.0 for i in range(len(counts))]
        per_block = torch.tensor(blocks, device="cuda")
        s["decay"] = torch.repeat_interleave(torch.tensor(decay, device="cuda"), per_block)[:, None]
        size = torch.empty(len(counts), device="cuda").log_normal_(-7.0, 1.0, generator=gen)
        size = torch.repeat_interleave(size, per_block)[:, None]
        scale = 1024.0 if case["type"] == "f16" else 1.0   # the loss scale of half-precision gradients

        def normal():
            x = torch.empty(nb * BLOCK, device="cuda").normal_(generator=gen)
            return (x * inside).view(nb, BLOCK)

        s["g"] = [(normal() * (size * scale)).to(TYPES[case["type"]]).view(-1) for _ in range(case["ranks"])]
        s["w"] = (normal() * 0.02).view(-1)
        s["inv_scale"] = 1.0 / (scale * case["ranks"])
        m = normal() * (size * 0.3)
        r = normal().abs().add_(0.05).mul_(size) * inside.view(nb, BLOCK)
        if case["bits"] == 8:
            s["m"], s["sm"] = _to_e4m3(m, False)
            s["v"], s["sv"] = _to_e4m3(r, True)
            s["m"], s["v"] = s["m"].view(-1), s["v"].view(-1)
            s["scales"] = torch.cat([s.pop("sm").view(-1), s.pop("sv").view(-1)])
        else:
            s["m"], s["v"] = m.view(-1), (r * r).view(-1)
        s["w16"] = None if case["copy"] == "none" else torch.zeros(nb * BLOCK, device="cuda", dtype=TYPES[case["copy"]])
        s["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["step"] = 100
        if own:
            from coconet_amd import capi
            s["plan"] = capi.AdamWPlan(counts, decay=decay, bits=case["bits"])
            cut = lambda x: [x[o:o + c] for o, c in zip(starts, counts)]  # noqa: E731
            s["tables"] = s["plan"].tables([cut(g) for g in s["g"]], cut(s["w"]), None if s["w16"] is None else cut(s["w16"]))
        return s
    t, M, K, N, pad = TYPES[case["type"]], case["M"], case["K"], case["N"], case["pad"]
    s["X"] = _rows(gen, M, K, pad, 1.0, t)
    s["W"] = _rows(gen, K, N, pad, 0.02, t)
    if case["op"] == "linear":
        s["b"] = torch.empty(N, device="cuda").normal_(0.0, 0.1, generator=gen) if case["bias"] else None
        s["R"] = _rows(gen, M, N, pad, 1.0, t) if case["resid"] else None
        s["Y"] = torch.empty(M, N, device="cuda", dtype=t)
        s["pre"] = torch.empty(M, N, device="cuda", dtype=t) if case["keep"] else None
    else:
        s["dY"] = _rows(gen, M, N, pad, 0.01, t)
        s["pre"] = None if case["act"] == "none" else _rows(gen, M, N, pad, 1.0, t)
        s["dX"] = torch.empty(M, K, device="cuda", dtype=t)
        s["sum"] = case["grad"] == "f32"
        s["dW"] = torch.empty(K, N, device="cuda", dtype=TYPES[case["grad"]])
        s["db"] = torch.empty(N, device="cuda")
        if s["sum"]:
            s["dW"].normal_(0.0, 0.5, generator=gen)
            s["db"].normal_(0.0, 0.5, generator=gen)
    if own:
        from coconet_amd import capi
        s["plan"] = capi.LinearPlan(M, N, K)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0.0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    if act == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        return e * (1.0 + z * (1.0 - e))
    return torch.ones_like(z)


def _to_e4m3(x, keep_above_zero):
    """x [blocks x BLOCK] as e4m3 values and the scale of each block [blocks x 1]."""
    scale = x.abs().amax(1, keepdim=True) / E4M3_MAX
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    if keep_above_zero:
        y = torch.where(x > 0, y.clamp_min(E4M3_TINY), y)
    return y.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _adamw(s, g, w, m, v, decay, step, flag):
    """One step on arrays of any float type: new w, m, v.  Elements whose gradient is not finite stay as they are."""
    bad = ~torch.isfinite(g)
    flag.copy_(bad.any())
    m2 = BETA1 * m + (1.0 - BETA1) * g
    v2 = BETA2 * v + (1.0 - BETA2) * g * g
    update = (m2 / (1.0 - BETA1 ** step)) / (torch.sqrt(v2 / (1.0 - BETA2 ** step)) + EPS)
    w2 = w * (1.0 - LR * WD * decay) - LR * update
    return torch.where(bad, w, w2), torch.where(bad, m, m2), torch.where(bad, v, v2)


def _plain_adamw(s):
    nb = s["w"].numel() // BLOCK
    g = s["g"][0].float()
    for x in s["g"][1:]:
        g = g + x.float()
    g = (g * s["inv_scale"]).view(nb, BLOCK)
    m, v = s["m"].float().view(nb, BLOCK), s["v"].float().view(nb, BLOCK)
    if s["bits"] == 8:
        sm, sv = s["scales"].view(2, nb, 1)
        m, v = m * sm, (v * sv) ** 2
    w, m, v = _adamw(s, g, s["w"].view(nb, BLOCK), m, v, s["decay"], s["step"], s["flag"])
    s["w"].copy_(w.view(-1))
    if s["w16"] is not None:
        s["w16"].copy_(w.view(-1))
    if s["bits"] == 8:
        m, sm = _to_e4m3(m, False)
        v, sv = _to_e4m3(torch.sqrt(v), True)
        s["scales"].copy_(torch.cat([sm.view(-1), sv.view(-1)]))
    s["m"].copy_(m.view(-1))
    s["v"].copy_(v.view(-1))


def _plain_linear(s):
    z = s["X"].float() @ s["W"].float()
    if s["b"] is not None:
        z = z + s["b"]
    if s["pre"] is not None:
        s["pre"].copy_(z)
    y = _act(z, s["act"])
    if s["R"] is not None:
        y = y + s["R"].float()
    s["Y"].copy_(y)


def _plain_backward(s):
    dz = s["dY"].float()
    if s["pre"] is not None:
        dz = dz * _act_slope(s["pre"].float(), s["act"])
    s["dX"].copy_(dz @ s["W"].float().t())
    dw, db = s["X"].float().t() @ dz, dz.sum(0)
    if s["sum"]:
        dw, db = s["dW"] + dw, s["db"] + db
    s["dW"].copy_(dw)
    s["db"].copy_(db)


# ---- the library's calls ---------------------------------------------------------------------------------------------
def _own_adamw(s):
    from coconet_amd import capi
    s["plan"].step(s["tables"], s["m"], s["v"], LR, BETA1, BETA2, EPS, WD, s["step"], scales=s.get("scales"), g_type=s["type"],
                   w16_type="bf16" if s["copy"] == "none" else s["copy"], inv_scale=s["inv_scale"], overflow_flag=s["flag"],
                   stream=capi.current_stream())


def _own_linear(s):
    from coconet_amd import capi
    s["plan"].forward(s["X"], s["W"], s["b"], s["R"], s["Y"], s["M"], s["N"], s["K"], act=s["act"], pre=s["pre"], half=s["type"] == "f16",
                      ldx=s["X"].stride(0), ldw=s["W"].stride(0), ldr=s["R"].stride(0) if s["R"] is not None else 0, stream=capi.current_stream())


def _own_backward(s):
    from coconet_amd import capi
    s["plan"].backward(s["dY"], s["pre"], s["X"], s["W"], s["dX"], s["dW"], s["db"], s["M"], s["N"], s["K"], act=s["act"], half=s["type"] == "f16",
                       dw_f32=s["sum"], accumulate=s["sum"], lddy=s["dY"].stride(0), ldp=s["pre"].stride(0) if s["pre"] is not None else 0,
                       ldx=s["X"].stride(0), ldw=s["W"].stride(0), stream=capi.current_stream())


def run(state):
    s = state
    (_own_adamw if own else _plain_adamw)(s) if s["op"] == "adamw" else \
        (_own_linear if own else _plain_linear)(s) if s["op"] == "linear" else (_own_backward if own else _plain_backward)(s)
    keys = {"adamw": ("w", "w16", "m", "v", "scales", "flag"), "linear": ("Y", "pre"), "backward": ("dX", "dW", "db")}[s["op"]]
    return {k: s[k] for k in keys if s.get(k) is not None}


# ---- what one pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        n = sum(_counts(case))
        g = case["ranks"] * (4 if case["type"] == "f32" else 2)
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (g + 8 + moments + (0 if case["copy"] == "none" else 2)), "flops": n * 16}
    M, K, N = case["M"], case["K"], case["N"]
    if case["op"] == "linear":
        outs = 1 + int(case["keep"]) + int(case["resid"])
        return {"bytes": 2 * (M * K + K * N + M * N * outs) + 4 * N * int(case["bias"]), "flops": 2 * M * N * K}
    grads = {"f32": 8}.get(case["grad"], 2)
    return {"bytes": 2 * (2 * M * K + K * N + M * N * (1 if case["act"] == "none" else 2)) + grads * K * N + 4 * N, "flops": 4 * M * N * K}


# ---- in 64 bits, from the definitions --------------------------------------------------------------------------------
def _slope64(z, act):
    """The derivative of each activation, through autograd of its definition."""
    z = z.clone().requires_grad_(True)
    phi = torch.special.ndtr(z)
    y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * phi,
         "gelu_tanh": lambda: z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)),
         "silu": lambda: z * torch.sigmoid(z)}[act]()
    y.backward(torch.ones_like(y))
    return y.detach(), z.grad


def _e4m3_64(x, keep_above_zero):
    """x / scale rounded to the nearest e4m3 value (ties to even), in 64 bits, and the scale."""
    scale = x.abs().amax(1, keepdim=True) / E4M3_MAX
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(e - 4, min=-9))   # 3 bits behind the leading one; below 2^-6 even steps
    q = torch.round(y / step) * step
    if keep_above_zero:
        q = torch.where((x > 0) & (q < E4M3_TINY), torch.full_like(q, E4M3_TINY), q)
    return q, scale


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda x: x.to(torch.float64)  # noqa: E731
    if case["op"] == "adamw":
        nb = s["w"].numel() // BLOCK
        g = torch.stack([d(x) for x in s["g"]]).sum(0).view(nb, BLOCK) * s["inv_scale"]
        m, v, w = d(s["m"]).view(nb, BLOCK), d(s["v"]).view(nb, BLOCK), d(s["w"]).view(nb, BLOCK)
        if case["bits"] == 8:
            sm, sv = d(s["scales"]).view(2, nb, 1)
            m, v = m * sm, (v * sv).square()
        m += (1.0 - BETA1) * (g - m)
        v += (1.0 - BETA2) * (g.square() - v)
        mhat, vhat = m / (1.0 - BETA1 ** s["step"]), v / (1.0 - BETA2 ** s["step"])
        w = w - LR * (mhat / (vhat.sqrt() + EPS) + WD * d(s["decay"]) * w)
        out = {"w": w.view(-1), "flag": s["flag"]}
        if case["copy"] != "none":
            out["w16"] = w.view(-1)
        if case["bits"] == 8:
            m, sm = _e4m3_64(m, False)
            v, sv = _e4m3_64(v.sqrt(), True)
            out["scales"] = torch.cat([sm.view(-1), sv.view(-1)])
        out["m"], out["v"] = m.view(-1), v.view(-1)
        return out
    X, W = d(s["X"]), d(s["W"])
    if case["op"] == "linear":
        z = X @ W
        if s["b"] is not None:
            z += d(s["b"])
        y = _slope64(z, case["act"])[0]
        out = {"Y": y if s["R"] is None else y + d(s["R"])}
        if s["pre"] is not None:
            out["pre"] = z
        return out
    dz = d(s["dY"])
    if s["pre"] is not None:
        dz = dz * _slope64(d(s["pre"]), case["act"])[1]
    dw, db = X.t() @ dz, dz.sum(0)
    if s["sum"]:
        dw, db = dw + d(s["dW"]), db + d(s["db"])
    return {"dX": dz @ W.t(), "dW": dw, "db": db}
