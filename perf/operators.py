"""What is measured of the decoder-side operators: residual + root-mean-square norm with an 8-bit output, rotary positions at given
(far, scaled) places, and attention with a sliding window and sinks.  `run` computes the plain form in elementary torch operations, or, where
`own` is set, makes the calls a user of the package makes."""
import math

import numpy as np
import torch

own = False

BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one sequence between two W8A8 linears: launch latency
        dict(name="norm_step_fp8", op="norm", rows=1, width=4096, quant="fp8"),
        # a long prompt's rows in front of an fp8 linear
        dict(name="norm_prompt_fp8", op="norm", rows=16384, width=5120, quant="fp8"),
        # a ragged number of rows in front of an int8 linear
        dict(name="norm_ragged_int8", op="norm", rows=1023, width=1536, quant="int8"),
        # bf16 output (unquantised linears), an odd number of rows
        dict(name="norm_rows_bf16", op="norm", rows=4099, width=3584, quant="none"),
        # one token each of 32 sequences, far behind the trained length
        dict(name="rope_step", op="rope", batch=32, seq=1, q_heads=32, kv_heads=8, head=128, rot=128, neox=True, scaling="yarn",
             factor=16.0, base=1000000.0, original=8192, far=131072),
        # a long prompt, half layout, shared key heads
        dict(name="rope_prompt", op="rope", batch=1, seq=16384, q_heads=32, kv_heads=8, head=128, rot=128, neox=True, scaling="wavelength",
             factor=8.0, base=500000.0, original=8192, far=16384),
        # interleaved layout, half of the head rotated, an odd length
        dict(name="rope_partial", op="rope", batch=3, seq=1371, q_heads=24, kv_heads=24, head=64, rot=32, neox=False, scaling="ntk",
             factor=4.0, base=10000.0, original=2048, far=8192),
        # one token each of 16 sequences over their caches
        dict(name="window_step", op="window", batch=16, seq=1, past=16383, q_heads=32, kv_heads=8, head=128, window=4096, sinks=4, ragged=True),
        # one token of one sequence, short window: launch latency
        dict(name="window_step_short", op="window", batch=1, seq=1, past=299, q_heads=24, kv_heads=24, head=64, window=128, sinks=1, ragged=False),
        # a long prompt
        dict(name="window_prompt", op="window", batch=1, seq=16384, past=0, q_heads=32, kv_heads=8, head=128, window=4096, sinks=4, ragged=False),
        # a padded batch of prompts of different lengths
        dict(name="window_batch", op="window", batch=4, seq=1531, past=0, q_heads=24, kv_heads=24, head=64, window=512, sinks=64, ragged=True),
        # a chunk of a prompt behind what the cache holds already
        dict(name="window_chunk", op="window", batch=2, seq=512, past=7900, q_heads=28, kv_heads=4, head=128, window=2048, sinks=16, ragged=True),
    ]


def _spread(rng, lo, hi):
    """A whole number, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "rope", "window"))
    if op == "norm":
        width = 8 * _spread(rng, 8, 1024)
        if rng.random() < 0.2:
            width += rng.randint(1, 7)
        rows = _spread(rng, 1, min(16384, 12288 * 5120 // width))
        return dict(op=op, rows=rows, width=width, quant=rng.choice(("none", "fp8", "int8")))
    if op == "rope":
        head = rng.choice((32, 64, 80, 96, 128, 256))
        rot = rng.choice((head, head, head // 2, head // 4))
        kv_heads = rng.choice((1, 2, 4, 8, 24))
        q_heads = kv_heads * rng.choice((1, 2, 4))
        seq = 1 if rng.random() < 0.4 else _spread(rng, 2, 16384)
        most = 16384 * 32 * 128 // (seq * (q_heads + kv_heads) * head)
        batch = _spread(rng, 1, max(1, min(64, most)))
        return dict(op=op, batch=batch, seq=seq, q_heads=q_heads, kv_heads=kv_heads, head=head, rot=rot, neox=rng.random() < 0.5,
                    scaling=rng.choice(("none", "linear", "ntk", "yarn", "wavelength")), factor=rng.choice((2.0, 4.0, 16.0)),
                    base=rng.choice((10000.0, 500000.0, 1000000.0)), original=rng.choice((2048, 4096, 8192)),
                    far=_spread(rng, 32768, 1 << 20))
    kv_heads = rng.choice((1, 2, 8, 24))
    q_heads = kv_heads * rng.choice((1, 2, 4, 7))
    head = rng.choice((64, 128))
    seq = 1 if rng.random() < 0.4 else _spread(rng, 2, 8192)
    past = _spread(rng, 1, 16384) if seq == 1 or rng.random() < 0.5 else 0
    most = min(32 * 16384 * 16384 // (8 * q_heads * seq * (seq + past)), 16 * 16384 * 8 * 128 // ((seq + past) * kv_heads * head))
    batch = _spread(rng, 1, max(1, min(32, most)))
    return dict(op=op, batch=batch, seq=seq, past=past, q_heads=q_heads, kv_heads=kv_heads, head=head, window=_spread(rng, 16, 8192),
                sinks=rng.choice((0, 1, 4, 16, 64, 130)), ragged=rng.random() < 0.6)


def _lengths(case):
    """Tokens of each sequence that are queries of this call, and all its tokens (the queries are the last of them)."""
    B, seq, past = case["batch"], case["seq"], case["past"]
    if not case["ragged"]:
        return [seq] * B, [seq + past] * B
    q = [seq - b * (seq - 1) // (2 * B) for b in range(B)]
    return q, [n + past - (B - 1 - b) * past // (2 * B) for b, n in enumerate(q)]


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    state = dict(case=case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # a residual stream has a few channels far over the others, and grows over the layers; the layer's output is smaller
        channel = torch.where(torch.rand(width, generator=g, device="cuda") < 0.01, 20.0, 1.0)
        state["residual"] = (normal(rows, width) * channel * 2.0).to(BF16)
        state["x"] = (normal(rows, width) * channel * 0.5).to(BF16)
        state["weight"] = (1.0 + 0.2 * normal(width)).to(BF16)
        state["eps"] = 1e-6
        return state
    B, S, Hq, Hk, D = case["batch"], case["seq"], case["q_heads"], case["kv_heads"], case["head"]
    if case["op"] == "rope":
        # the fused projection's output, and each sequence's own place
        state["qkv"] = normal(B, S, (Hq + 2 * Hk) * D).to(BF16)
        first = torch.randint(0, max(1, case["far"] - S), (B, 1), generator=g, device="cuda")
        state["positions"] = first + torch.arange(S, device="cuda")
        state["frequencies"] = _plan(case)
        return state
    past = case["past"]
    q_lens, kv_lens = _lengths(case)
    # keys near the first tokens' direction and queries that look for it: the first tokens draw a good share of the weights
    toward = normal(1, 1, Hk, 1, D)
    state["query"] = (1.5 * normal(B, S, Hk, Hq // Hk, D) + 0.35 * toward).reshape(B, S, Hq * D).to(BF16)
    key = normal(B, S + past, Hk, D)
    key[:, :max(1, case["sinks"])] += toward[:, :, :, 0]
    state["key"] = key.reshape(B, S + past, Hk * D).to(BF16)
    state["value"] = (normal(B, S + past, Hk, D) + 0.5 * normal(1, 1, Hk, D)).reshape(B, S + past, Hk * D).to(BF16)
    state["q_lens"] = torch.tensor(q_lens, dtype=torch.int32, device="cuda") if case["ragged"] else None
    state["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device="cuda") if case["ragged"] else None
    return state


def _plan(case):
    """What a program makes once of a model's rotary settings."""
    kind = None if case["scaling"] == "none" else case["scaling"]
    if own:
        from fastdm_amd.layer.embeddings import RotaryFrequencies
        return RotaryFrequencies(case["rot"], base=case["base"], scaling=kind, factor=case["factor"], original_length=case["original"], device="cuda")
    d, base, s, original = case["rot"], case["base"], case["factor"], case["original"]
    if kind == "ntk":
        base = base * s ** (d / (d - 2))
    i = torch.arange(d // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / d)
    amplitude = 1.0
    if kind == "linear":
        f = f / s
    elif kind == "yarn":
        low = max(0, math.floor(d * math.log(original / (32.0 * 2.0 * math.pi)) / (2.0 * math.log(base))))
        high = min(d - 1, math.ceil(d * math.log(original / (1.0 * 2.0 * math.pi)) / (2.0 * math.log(base))))
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        f = f / s * ramp + f * (1.0 - ramp)
        amplitude = 0.1 * math.log(s) + 1.0
    elif kind == "wavelength":
        keep = ((original * f / (2.0 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f / s * (1.0 - keep) + f * keep
    return f.cuda(), amplitude


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    return _norm(state) if op == "norm" else _rope(state) if op == "rope" else _window(state)


def _norm(state):
    x, residual, weight, eps, quant = state["x"], state["residual"], state["weight"], state["eps"], state["case"]["quant"]
    if own:
        from fastdm_amd.kernel.fused import add_rms_norm
        if quant == "none":
            y, _, h = add_rms_norm(x, residual, weight, eps)
            return dict(sum=h, y=y)
        _, z, h = add_rms_norm(x, residual, weight, eps, quant=FP8 if quant == "fp8" else torch.int8)
        if quant == "fp8":
            return dict(sum=h, q=z.q, scale=z.scale)
        return dict(sum=h, q=torch.sub(z.q, z.azp, out=torch.empty_like(h)), scale=z.scale)
    h = (x.float() + residual.float()).to(BF16)          # the residual stream is kept in the activations' type, and normed as it is kept
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(1, keepdim=True) + eps) * weight.float()
    if quant == "none":
        return dict(sum=h, y=y.to(BF16))
    if quant == "fp8":
        scale = y.abs().amax(1, keepdim=True) / 448.0
        return dict(sum=h, q=(y / scale).clamp(-448.0, 448.0).to(FP8), scale=scale)
    low, high = y.amin(1, keepdim=True), y.amax(1, keepdim=True)
    scale = (high - low) / 255.0
    zero = -128.0 - torch.round(low / scale)
    q = torch.round(y / scale + zero).clamp(-128.0, 127.0)
    return dict(sum=h, q=(q - zero).to(BF16), scale=scale)     # steps of `scale` from zero: whole numbers of up to 256, exact in bf16


def _rope(state):
    case, qkv, positions = state["case"], state["qkv"], state["positions"]
    Hq, Hk, D, rot = case["q_heads"], case["kv_heads"], case["head"], case["rot"]
    if own:
        from fastdm_amd.kernel.operators_set import rotary_positions
        q, k = rotary_positions(qkv[..., :Hq * D], qkv[..., Hq * D:(Hq + Hk) * D], D, state["frequencies"], positions, is_neox=case["neox"])
        return dict(q=q, k=k)
    B, S = positions.shape
    f, amplitude = state["frequencies"]
    angle = positions.double()[..., None] * f
    c, s = (angle.cos() * amplitude).float()[:, :, None], (angle.sin() * amplitude).float()[:, :, None]
    x = qkv[..., :(Hq + Hk) * D].float().reshape(B, S, Hq + Hk, D)
    turned, rest = x[..., :rot], x[..., rot:]
    if case["neox"]:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    out = torch.cat((turned, rest), -1).to(BF16)
    return dict(q=out[:, :, :Hq].reshape(B, S, Hq * D), k=out[:, :, Hq:].reshape(B, S, Hk * D))


def _window(state):
    case, q, k, v, q_lens, kv_lens = state["case"], state["query"], state["key"], state["value"], state["q_lens"], state["kv_lens"]
    Hq, Hk, D = case["q_heads"], case["kv_heads"], case["head"]
    if own:
        from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention
        return window_scaled_dot_product_attention(q, k, v, Hq, Hk, D, case["window"], sinks=case["sinks"], q_lens=q_lens, kv_lens=kv_lens)
    B, S, L = q.shape[0], q.shape[1], k.shape[1]
    qn = torch.full((B,), S, device=q.device) if q_lens is None else q_lens.long()
    kn = torch.full((B,), L, device=q.device) if kv_lens is None else kv_lens.long()
    row, j = torch.arange(S, device=q.device)[None, :, None], torch.arange(L, device=q.device)[None, None, :]
    place = (kn - qn)[:, None, None] + row
    seen = (j <= place) & ((place - j < case["window"]) | (j < case["sinks"])) & (row < qn[:, None, None])
    qf = q.float().reshape(B, S, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, Hq // Hk * S, D)
    kf = k.float().reshape(B, L, Hk, D).permute(0, 2, 3, 1).contiguous()
    vf = v.float().reshape(B, L, Hk, D).transpose(1, 2).contiguous()
    p = torch.matmul(qf, kf).mul_(D ** -0.5).view(B, Hk, Hq // Hk, S, L)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min_(-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, Hq // Hk * S, L), vf).view(B, Hk, Hq // Hk, S, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))                # a row that sees nothing is zero
    return o.permute(0, 3, 1, 2, 4).reshape(B, S, Hq * D).to(BF16)


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        if case["quant"] == "none":
            return dict(bytes=n * 8 + 2 * case["width"], flops=6 * n)
        return dict(bytes=n * 7 + 2 * case["width"] + 4 * case["rows"], flops=8 * n)
    B, S, Hq, Hk, D = case["batch"], case["seq"], case["q_heads"], case["kv_heads"], case["head"]
    if case["op"] == "rope":
        n = B * S * (Hq + Hk)
        return dict(bytes=n * D * 4 + B * S * 8 + case["rot"] * 4, flops=3 * n * case["rot"])
    pairs = keys = rows = 0
    for qn, kn in zip(*_lengths(case)):
        n = np.arange(kn - qn, kn, dtype=np.int64) + 1                       # tokens up to each query, itself among them
        pairs += int((np.minimum(n, case["window"]) + np.minimum(case["sinks"], np.maximum(0, n - case["window"]))).sum())
        keys += min(kn, qn - 1 + case["window"] + case["sinks"])
        rows += qn
    return dict(bytes=2 * D * ((rows + B * S) * Hq + 2 * keys * Hk), flops=4 * pairs * Hq * D)


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        h64 = state["x"].double() + state["residual"].double()
        kept = h64.to(BF16).double()
        y = kept / ((kept ** 2).sum(1, keepdim=True) / case["width"] + state["eps"]).sqrt() * state["weight"].double()
        if case["quant"] == "none":
            return dict(sum=h64, y=y)
        if case["quant"] == "fp8":
            scale = y.abs().max(1, keepdim=True).values / 448
        else:
            scale = (y.max(1, keepdim=True).values - y.min(1, keepdim=True).values) / 255
            return dict(sum=h64, q=(y / scale).round(), scale=scale)         # whole steps by definition
        return dict(sum=h64, q=y / scale, scale=scale)
    if case["op"] == "rope":
        return _exact_rope(case, state)
    D, Hq, Hk, W, N = case["head"], case["q_heads"], case["kv_heads"], case["window"], case["sinks"]
    q, k, v = state["query"], state["key"], state["value"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (qn, kn) in enumerate(zip(*_lengths(case))):
        for r0 in range(0, qn, 512):
            r1 = min(qn, r0 + 512)
            p0, p1 = kn - qn + r0, kn - qn + r1                              # places of the chunk's rows: p0 .. p1 - 1
            near = max(0, p0 - W + 1)
            at = torch.cat((torch.arange(min(N, near)), torch.arange(near, p1))).to(q.device)
            place = torch.arange(p0, p1, device=q.device)[:, None]
            hidden = (at > place) | ((at <= place - W) & (at >= N))
            kk = k[b, at].double().view(-1, Hk, D).permute(1, 2, 0).contiguous()
            vv = v[b, at].double().view(-1, Hk, D).transpose(0, 1).contiguous()
            qq = q[b, r0:r1].double().view(r1 - r0, Hk, Hq // Hk, D)
            for h in range(Hq // Hk):
                w = torch.bmm(qq[:, :, h].transpose(0, 1).contiguous(), kk) / math.sqrt(D)
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                out[b, r0:r1].view(r1 - r0, Hk, Hq // Hk, D)[:, :, h] = torch.bmm(w, vv).transpose(0, 1)
    return out


def _exact_rope(case, state):
    B, S = state["positions"].shape
    Hq, Hk, D, d, s, L = case["q_heads"], case["kv_heads"], case["head"], case["rot"], case["factor"], case["original"]
    base = np.float64(case["base"]) * (s ** (d / (d - 2.0)) if case["scaling"] == "ntk" else 1.0)
    f, amplitude = [], 1.0
    for i in range(d // 2):
        plain = 1.0 / base ** (2.0 * i / d)
        if case["scaling"] == "linear":
            plain /= s
        elif case["scaling"] == "yarn":
            def turns_at(n):                                                  # the pair that turns n times within the trained length
                return d * np.log(L / (n * 2 * np.pi)) / (2 * np.log(base))
            low, high = max(np.floor(turns_at(32)), 0), min(np.ceil(turns_at(1)), d - 1)
            slow = np.clip((i - low) / (high - low if high > low else 1e-3), 0, 1)
            plain = plain * (1 - slow) + plain / s * slow
            amplitude = 1 + np.log(s) / 10
        elif case["scaling"] == "wavelength":
            length = 2 * np.pi / plain
            if length > L:
                plain /= s
            elif length > L / 4.0:
                mix = (L / length - 1) / 3
                plain = (1 - mix) * plain / s + mix * plain
        f.append(plain)
    angle = state["positions"].double()[:, :, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, float(amplitude)), angle)
    out = []
    for at, heads in ((0, Hq), (Hq * D, Hk)):
        x = state["qkv"][..., at:at + heads * D].double().reshape(B, S, heads, D)
        if case["neox"]:
            z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:d].contiguous()) * turn
            y = torch.cat((z.real, z.imag, x[..., d:]), -1)
        else:
            z = torch.view_as_complex(x[..., :d].reshape(B, S, heads, d // 2, 2).contiguous()) * turn
            y = torch.cat((torch.view_as_real(z).flatten(-2), x[..., d:]), -1)
        out.append(y.reshape(B, S, heads * D))
    return dict(q=out[0], k=out[1])
