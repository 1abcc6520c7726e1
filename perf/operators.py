"""What the 8-bit operators are measured on: the int8 linear layer with a scale for each token and output channel, and 8-bit
activation checkpoints (groups of 64 columns with a power-of-two scale) with the three places a backward pass reads one: LayerNorm,
GELU and a linear layer's weight gradient.

`own` False: the operators in elementary torch operations; True: the framework's kernels (climb_amd.rows8)."""
import math

import torch

own = False

GROUP = 64                  # columns that share a checkpoint scale
FLT_MIN = 2.0 ** -126
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # evaluation of one image-text pair: the pooled row through a 768 x 768 product (one token: latency)
        dict(name="linear_one_token", op="linear", M=1, K=768, N=768, x="bf16", y="bf16", epi="none"),
        # the VQA answer head for a batch of 64: 1536 features to 3129 answers in fp32 (an odd width)
        dict(name="linear_vqa_head", op="linear", M=64, K=1536, N=3129, x="f32", y="f32", epi="none"),
        # the encoder's MLP for 64 sequences of 192 rows: up-projection with GELU ...
        dict(name="linear_mlp_up", op="linear", M=12288, K=768, N=3072, x="bf16", y="bf16", epi="gelu"),
        # ... and down-projection added to the fp32 residual stream
        dict(name="linear_mlp_down", op="linear", M=12288, K=3072, N=768, x="bf16", y="f32", epi="resid"),
        # fine-tuning on one sequence of 185 tokens (40 text + class + 144 patches): the attention output projection's weight gradient
        dict(name="wgrad_one_sequence", op="wgrad", M=185, K=768, N=768, x="bf16"),
        # the answer head's second product at a batch of 64, kept in fp32
        dict(name="wgrad_vqa_head", op="wgrad", M=64, K=1536, N=3129, x="f32"),
        # the MLP's up-projection at the benchmark batch
        dict(name="wgrad_mlp_up", op="wgrad", M=12288, K=768, N=3072, x="bf16"),
        # a layer's LayerNorm on one sequence
        dict(name="layernorm_one_sequence", op="layernorm", M=185, C=768, y="bf16"),
        # the answer head's LayerNorm in fp32 at the batch of a replay step
        dict(name="layernorm_head_f32", op="layernorm", M=333, C=1536, y="f32"),
        # a layer's LayerNorm at the benchmark batch
        dict(name="layernorm_layer", op="layernorm", M=12288, C=768, y="bf16"),
        # the MLP's GELU on one sequence, and at the benchmark batch
        dict(name="gelu_one_sequence", op="gelu", M=185, C=3072, x="bf16"),
        dict(name="gelu_layer", op="gelu", M=12288, C=3072, x="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """linear: 1 .. 12288 tokens, widths 16 .. 3200, up to the MLP's 2 x 12288 x 768 x 3072 operations; checkpoints: 1 .. 12288 rows"""
    op = rng.choice(["linear", "wgrad", "layernorm", "gelu"])
    if op in ("linear", "wgrad"):
        while True:
            M, K, N = _log(rng, 1, 12288), _log(rng, 16, 3200), _log(rng, 16, 3200)
            if M * K * N <= 12288 * 768 * 3072:
                break
        if op == "wgrad":
            return dict(op=op, M=M, K=K, N=N, x=rng.choice(["bf16", "f32"]))
        epi = rng.choice(["none", "gelu", "resid"])
        return dict(op=op, M=M, K=K, N=N, x=rng.choice(["bf16", "f32"]), y="f32" if epi == "resid" else rng.choice(["bf16", "f32"]), epi=epi)
    if op == "layernorm":
        C = _log(rng, 32, 1536)
        return dict(op=op, M=_log(rng, 1, 12288 * 768 // max(C, 768)), C=C, y=rng.choice(["bf16", "f32"]))
    M, C = _log(rng, 1, 12288), _log(rng, 16, 3072)
    return dict(op=op, M=M, C=C, x="bf16" if M * C > 12288 * 1024 else rng.choice(["bf16", "f32"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)

    def rn(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def outliers(t):          # a few channels of a transformer's activations are tens of times the rest
        C = t.shape[1]
        t[:, torch.randint(0, C, (1 + C // 256,), generator=g, device="cuda")] *= 20.0
        return t

    op, M = case["op"], case["M"]
    st = dict(case=dict(case))
    if op == "linear":
        K, N = case["K"], case["N"]
        st["x"] = outliers(rn(M, K)).to(DT[case["x"]])
        w = rn(N, K, std=0.02)
        st["bias"] = rn(N, std=0.1)
        st["resid"] = rn(M, N) if case["epi"] == "resid" else None
        if own:          # the weights are laid out once and kept
            from climb_amd import rows8
            st["w"] = rows8.quantize_rows(w)
        else:
            st["w"] = _row_codes(w)
    elif op == "wgrad":
        st["x"] = outliers(rn(M, case["K"])).to(DT[case["x"]])
        st["dy"] = rn(M, case["N"], std=1e-3, dtype=torch.bfloat16)
    elif op == "layernorm":
        C, dt = case["C"], DT[case["y"]]
        st["x"] = outliers(rn(M, C))
        st["gamma"], st["beta"] = 1.0 + rn(C, std=0.1), rn(C, std=0.1)
        st["dy"], st["dres"] = rn(M, C, std=1e-3, dtype=dt), rn(M, C, std=1e-3)
    else:
        dt = DT[case["x"]]
        st["u"], st["da"] = rn(M, case["C"], std=1.5, dtype=dt), rn(M, case["C"], std=1e-3, dtype=dt)
    return st


# ----------------------------------------------------------------------------------------------------------- plain forms
def _row_codes(x):
    """(codes as fp32, scale): scale = amax / 127 rounded to fp32, codes = the true quotient rounded to even (both quotients in 64 bits:
    a scalar divisor is multiplied by its reciprocal in 32, and the codes' quotients lie next to halves)"""
    x = x.float()
    amax = x.abs().amax(1, keepdim=True)
    s = torch.where(torch.isfinite(amax), (amax.double() / 127.0).float().clamp(min=FLT_MIN), torch.full_like(amax, float("nan")))
    q = torch.nan_to_num(torch.round(x.double() / s.double()), nan=0.0).float()
    return q, s[:, 0]


def _checkpoint(x):
    """the values an 8-bit checkpoint of x stands for: per group of 64 columns, multiples of the smallest power of two that keeps |code| <= 127"""
    x = x.float()
    M, C = x.shape
    G = -(-C // GROUP)
    xp = torch.zeros(M, G * GROUP, device=x.device)
    xp[:, :C] = x
    xg = xp.view(M, G, GROUP)
    amax = xg.abs().amax(2, keepdim=True)
    m, k = torch.frexp(amax)                                    # amax = m 2^k, m in [0.5, 1); 127 2^e = 0.9921875 2^(e + 7)
    e = (k - 7 + (m > 0.9921875).to(k.dtype)).clamp(min=-126)
    e = torch.where(amax == 0, torch.full_like(e, -126), e)
    step = torch.ldexp(torch.ones_like(amax), e)
    v = torch.where(torch.isfinite(amax), torch.round(xg / step) * step, torch.full_like(xg, float("nan")))
    return v.reshape(M, G * GROUP)[:, :C]


def _phi_parts(u):
    return 0.5 * torch.special.erfc(u * -0.7071067811865476), torch.exp(-0.5 * u * u) * 0.3989422804014327


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "linear":
        q, s = _row_codes(st["x"])
        wq, ws = st["w"]
        y = (q @ wq.t()) * s[:, None] * ws[None, :] + st["bias"]
        if case["epi"] == "gelu":
            y = y * _phi_parts(y)[0]
        elif case["epi"] == "resid":
            y = y + st["resid"]
        return y.to(DT[case["y"]])
    if op == "wgrad":
        v, dy = _checkpoint(st["x"]), st["dy"].float()
        return dy.t() @ v, dy.sum(0)
    if op == "layernorm":
        x, gamma, dy = st["x"], st["gamma"], st["dy"].float()
        mean = x.mean(1, keepdim=True)
        rstd = torch.rsqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-12)
        y = (x - mean) * rstd * gamma + st["beta"]
        xh = (_checkpoint(x) - mean) * rstd                     # the backward sees the checkpoint
        G = dy * gamma
        dx = st["dres"] + rstd * (G - G.mean(1, keepdim=True) - xh * (G * xh).mean(1, keepdim=True))
        return y.to(DT[case["y"]]), dx, (dy * xh).sum(0), dy.sum(0)
    dt = DT[case["x"]]
    u, da = st["u"].float(), st["da"].float()
    a = u * _phi_parts(u)[0]
    v = _checkpoint(st["u"])
    cdf, pdf = _phi_parts(v)
    return a.to(dt), (da * (cdf + v * pdf)).to(dt), (v * cdf).to(dt)


# -------------------------------------------------------------------------------------------------------------- kernels
def _run_own(st):
    from climb_amd import rows8
    case = st["case"]
    op = case["op"]
    if op == "linear":
        return rows8.linear_i8(st["x"], st["w"], st["bias"], epi=case["epi"], resid=st["resid"], out_dtype=DT[case["y"]])
    if op == "wgrad":                       # the forward keeps x in 8 bits, the backward reads it
        ck = rows8.checkpoint_save(st["x"])
        return rows8.weight_grad(st["dy"], ck)
    if op == "layernorm":
        y, ck = rows8.layernorm_fwd(st["x"], st["gamma"], st["beta"], 1e-12, out_dtype=DT[case["y"]])
        dx, dgamma, dbeta = rows8.layernorm_bwd(st["dy"], ck, st["gamma"], dres=st["dres"])
        return y, dx, dgamma, dbeta
    a, ck = rows8.gelu_fwd(st["u"])
    du, a2 = rows8.gelu_bwd(st["da"], ck, recompute=True)
    return a, du, a2


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    M = case["M"]
    size = {"f32": 4, "bf16": 2}
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        b = M * K * size[case["x"]] + N * K + 8 * N + M * N * size[case["y"]] + (4 * M * N if case["epi"] == "resid" else 0)
        return {"bytes": b, "flops": 2 * M * N * K}
    if case["op"] == "wgrad":               # the codes are written by the forward and read by the backward: that is what a checkpoint is
        K, N = case["K"], case["N"]
        codes = M * K + M * (-(-K // GROUP))
        return {"bytes": M * K * size[case["x"]] + 2 * codes + 2 * M * N + 4 * N * K + 4 * N, "flops": 2 * M * N * K}
    C = case["C"]
    codes = M * C + M * (-(-C // GROUP))
    if case["op"] == "layernorm":
        s = size[case["y"]]
        return {"bytes": M * C * (4 + s + s + 4 + 4) + 2 * codes + 16 * C + 16 * M, "flops": 24 * M * C}
    return {"bytes": M * C * 5 * size[case["x"]] + 2 * codes, "flops": 50 * M * C}


# ----------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    global own
    was, own = own, False          # the same inputs, and the weights' codes of this file
    try:
        st = prepare(case, seed)
        op = case["op"]
        if op == "linear":
            return _exact_linear(case, st)
        if op == "wgrad":
            v, dy = _values64(st["x"]), st["dy"].double()
            return torch.mm(dy.t().contiguous(), v), torch.mm(torch.ones(1, dy.shape[0], device=dy.device, dtype=torch.float64), dy)[0]
        if op == "layernorm":
            x, dy, C = st["x"].double(), st["dy"].double(), case["C"]
            mu = x.sum(1) / C
            inv = 1.0 / torch.sqrt((x * x).sum(1) / C - mu * mu + 1e-12)
            y = (x - mu[:, None]) * inv[:, None] * st["gamma"].double() + st["beta"].double()
            n = (_values64(st["x"]) - mu[:, None]) * inv[:, None]
            h = dy * st["gamma"].double()
            m0, m1 = h.sum(1) / C, (h * n).sum(1) / C
            return y, st["dres"].double() + inv[:, None] * (h - m0[:, None] - n * m1[:, None]), (n * dy).sum(0), dy.sum(0)
        u, v, da = st["u"].double(), _values64(st["u"]), st["da"].double()
        return u * _ndtr64(u), da * (_ndtr64(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)), v * _ndtr64(v)
    finally:
        own = was


def _ndtr64(t):
    return torch.special.erfc(-t / math.sqrt(2.0)) / 2


def _codes64(t):
    """q and s of rows: the stored scale is an fp32 number, the code its nearest multiple"""
    t = t.double()
    s = torch.clamp((t.abs().max(dim=1).values / 127).float(), min=FLT_MIN).double()
    return torch.round(t / s[:, None]), s


def _values64(t):
    t = t.double()
    parts = []
    for c in range(0, t.shape[1], GROUP):
        p = t[:, c:c + GROUP]
        top = p.abs().max(dim=1, keepdim=True).values
        step = torch.exp2(torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -140) / 127.0)).clamp(min=-126))
        step = torch.where(step / 2 * 127 >= top, torch.clamp(step / 2, min=FLT_MIN), step)      # log2 next to a whole number
        step = torch.where(step * 127 < top, step * 2, step)
        parts.append(torch.round(p / step) * step)
    return torch.cat(parts, 1)


def _exact_linear(case, st):
    q, s = _codes64(st["x"])
    wq, ws = st["w"][0].double(), st["w"][1].double()
    y = torch.mm(q, wq.t().contiguous()) * torch.outer(s, ws) + st["bias"].double()
    if case["epi"] == "gelu":
        return y * _ndtr64(y)
    return y + st["resid"].double() if case["epi"] == "resid" else y
