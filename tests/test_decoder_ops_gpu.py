"""GPU: the decoder-side operators (add_rms_norm, rotary_positions, window_scaled_dot_product_attention) against plain 64-bit implementations.

Tolerances are half a step of the output's type relative to the value (bf16 2^-8, e4m3 2^-4, int8 half a scale), plus what the fp32 arithmetic in
front of that rounding can be off by, derived at each check."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
HALF_STEP = 2.0 ** -8          # of a bf16 value


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(BF16)


def assert_within(got, want, tol, what):
    """|got - want| <= tol element by element (want, tol in 64 bits)."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - tol
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.numel()} beyond, worst by {over.max().item():.3g}"


# ================================================================================================ add_rms_norm
def norm64(x, residual, weight, eps):
    h = x.double() if residual is None else (x.float() + residual.float()).to(BF16).double()      # (the fp32 sum of two bf16, rounded: what the stream keeps)
    return h, h * weight.double() / (h.square().mean(1, keepdim=True) + eps).sqrt()


def check_norm(y64, width, out, qz, quant):
    # fp32 in front of the rounding: `width` products summed over at most 1024 lanes and a tree (each step 2^-24, at most 64 + 16 of them in a row for
    # width 65536), square root, division, two products: under 100 * 2^-24 of the value
    rel = 100 * 2.0 ** -24
    if quant is None:
        assert_within(out, y64, y64.abs() * (HALF_STEP + rel), "y")
        return
    scale = qz.scale.double()
    if quant == FP8:
        want = y64.abs().amax(1, keepdim=True).clamp_min(1e-12) / 448.0
        assert ((scale - want).abs() <= want * 2 * rel).all()
        # e4m3: half a step is 2^-4 of the value, or 2^-10 under the smallest normal number
        assert_within(qz.q.double() * scale, y64, torch.maximum(y64.abs() * 2.0 ** -4, 2.0 ** -10 * want) * (1 + 4 * rel) + y64.abs() * 4 * rel, "e4m3")
        return
    low, high = y64.amin(1, keepdim=True), y64.amax(1, keepdim=True)
    size = torch.maximum(low.abs(), high.abs())
    want = torch.maximum(torch.maximum(high - low, size / 16), torch.full_like(size, 1e-12)) / 255.0
    assert ((scale - want).abs() <= 4 * rel * size / 255.0 + want * rel).all()      # (the spread is a difference: its error goes by the values' size)
    # half a step, plus the fp32 error of y / scale + zero point: |y| / scale <= 16 * 255, so a few 2^-24 of 4080 + 4080 steps
    assert_within((qz.q.double() - qz.azp.double()) * scale, y64, scale * (0.5 + 2.0 ** -8) + y64.abs() * 4 * rel, "int8")


@pytest.mark.parametrize("quant", [None, FP8, torch.int8])
@pytest.mark.parametrize("rows,width", [(1, 4096), (3, 8), (5, 1), (7, 13), (33, 512), (2, 520), (129, 1536), (17, 2048), (9, 3584), (4, 5120), (6, 6152),
                                        (3, 8192), (2, 8200), (2, 16384), (1, 30001), (1, 65536), (2, 65529), (5, 1003)])
def test_add_rms_norm(rows, width, quant):
    from fastdm_amd.kernel.fused import add_rms_norm
    g = gen(rows * 100000 + width)
    x, residual = randn(g, rows, width), randn(g, rows, width, scale=4.0)
    weight = (1 + 0.3 * torch.randn(width, generator=g, device="cuda")).to(BF16)
    for res in (residual, None):
        out, qz, h = add_rms_norm(x, res, weight, 1e-6, quant=quant)
        h64, y64 = norm64(x, res, weight, 1e-6)
        assert (h is None) == (res is None)
        if h is not None:
            assert torch.equal(h.double(), h64)
        check_norm(y64, width, out, qz, quant)


@pytest.mark.parametrize("quant", [None, FP8, torch.int8])
@pytest.mark.parametrize("width,wide,at", [(1536, 4608, 1536), (1000, 1500, 3), (72, 77, 1)])
def test_add_rms_norm_on_slices_and_in_place(width, wide, at, quant):
    """Rows that are column slices at aligned and odd places; the sum written over the residual, over x, and into a slice whose neighbours stay."""
    from fastdm_amd.kernel.fused import add_rms_norm
    g = gen(width + at)
    wx, wr = randn(g, 21, wide), randn(g, 21, wide)
    weight = randn(g, width)
    x, r = wx[:, at:at + width], wr[:, at:at + width]
    h64, y64 = norm64(x, r, weight, 1e-5)
    for into in ("new", "residual", "x", "slice"):
        bx, br, bo = wx.clone(), wr.clone(), randn(gen(3), 21, wide)
        before = {"residual": br, "x": bx, "slice": bo}.get(into)
        kept = None if before is None else before.clone()
        dst = None if before is None else before[:, at:at + width]
        out, qz, h = add_rms_norm(bx[:, at:at + width], br[:, at:at + width], weight, 1e-5, quant=quant, residual_out=dst)
        assert torch.equal(h.double(), h64)
        check_norm(y64, width, out, qz, quant)
        if before is not None:
            assert torch.equal(before[:, :at], kept[:, :at]) and torch.equal(before[:, at + width:], kept[:, at + width:])


def test_add_rms_norm_rows_of_one_value_of_zeros_and_of_nan():
    from fastdm_amd.kernel.fused import add_rms_norm
    width = 640
    x = torch.zeros(6, width, device="cuda", dtype=BF16)
    x[1] = 3.0                      # one value
    x[2, 5] = 1e-30                 # squares under fp32's range: y = 1e-30 / sqrt(eps)
    x[3] = torch.linspace(2.0, 2.05, width, device="cuda").to(BF16)
    x[4, 7] = float("nan")
    x[5, 7] = float("inf")
    weight = torch.ones(width, device="cuda", dtype=BF16)
    for quant in (None, FP8, torch.int8):
        out, qz, _ = add_rms_norm(x, None, weight, 1e-6, quant=quant)
        y64 = norm64(x, None, weight, 1e-6)[1]
        check_norm(y64[:4], width, None if out is None else out[:4], None if qz is None else type(qz)(qz.q[:4], qz.scale[:4], None if qz.azp is None else qz.azp[:4]), quant)
        if quant is None:
            assert torch.isnan(out[4]).all() and torch.isnan(out[5, 7])
        else:
            assert torch.isnan(qz.scale[4:]).all() and torch.isfinite(qz.scale[:4]).all()
        if quant == FP8:
            assert torch.isnan(qz.q[4:].float()).all()


def test_add_rms_norm_of_no_rows_and_on_another_stream():
    from fastdm_amd.kernel.fused import add_rms_norm
    weight = torch.ones(64, device="cuda", dtype=BF16)
    out, _, h = add_rms_norm(torch.empty(0, 64, device="cuda", dtype=BF16), torch.empty(0, 64, device="cuda", dtype=BF16), weight, 1e-6)
    assert out.shape == h.shape == (0, 64)
    x = randn(gen(1), 500, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = add_rms_norm(x, x, weight, 1e-6)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, add_rms_norm(x, x, weight, 1e-6)[0])


# ================================================================================================ rotary_positions
def rope64(x, head, freqs, positions, is_neox):
    B, S, W = x.shape
    rot = freqs.rotary_dim
    theta = torch.tensor(freqs.theta, dtype=torch.float64, device=x.device)
    angle = positions.double().expand(B, S)[:, :, None, None] * theta
    c, s = angle.cos() * freqs.amplitude, angle.sin() * freqs.amplitude
    x = x.double().reshape(B, S, W // head, head)
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if is_neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = a * c - b * s, b * c + a * s
    turned = torch.cat((u, v), -1) if is_neox else torch.stack((u, v), -1).flatten(-2)
    size = (a.abs() + b.abs()) * freqs.amplitude
    size = torch.cat((size, size), -1) if is_neox else torch.stack((size, size), -1).flatten(-2)
    out = torch.cat((turned, x[..., rot:]), -1)
    # the fraction of a turn in fp32 (at most 1/2: off by 2^-26 turns = 2 pi 2^-26 rad), sine and cosine 2^-23, their scaling, two products and a sum: under
    # 2^-20 of |a| + |b|; the 64-bit angles agree to 2^-50 * 2^21 turns
    tol = torch.cat((turned.abs() * HALF_STEP + size * 2.0 ** -20, torch.zeros_like(x[..., rot:])), -1)
    return out.reshape(B, S, W), tol.reshape(B, S, W)


@pytest.mark.parametrize("is_neox", [False, True])
@pytest.mark.parametrize("head,rot", [(128, 128), (64, 32), (64, 64), (80, 20), (96, 24), (256, 256), (256, 64), (10, 6), (7, 2), (128, 12), (8, 8), (2, 2), (1024, 16), (520, 250)])
@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 4, 1), (3, 37, 8, 2), (2, 5, 1, 1)])
def test_rotary_positions(B, S, Hq, Hk, head, rot, is_neox):
    from fastdm_amd.kernel.operators_set import rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    g = gen(B * 1000 + S + head + rot)
    q, k = randn(g, B, S, Hq * head), randn(g, B, S, Hk * head)
    freqs = RotaryFrequencies(rot, base=500000.0, scaling="yarn" if rot > 2 else None, factor=4.0, original_length=4096, device="cuda")
    far = torch.randint(0, 1 << 20, (B, S), generator=g, device="cuda")
    for positions in (None, far, far.int(), far[0], -far):
        qo, ko = rotary_positions(q, k, head, freqs, positions, is_neox=is_neox)
        at = torch.arange(S, device="cuda") if positions is None else positions
        for got, x in ((qo, q), (ko, k)):
            want, tol = rope64(x, head, freqs, at, is_neox)
            assert_within(got, want, tol, "rotary")


@pytest.mark.parametrize("is_neox", [False, True])
@pytest.mark.parametrize("head,rot,off", [(64, 64, 0), (64, 32, 3), (128, 96, 8), (96, 40, 4), (64, 16, 2)])
def test_rotary_positions_strided_in_place_and_into_a_cache(head, rot, off, is_neox):
    """Slices of a fused projection at places of every alignment, in place, and the key written into a slice of a cache; the neighbours stay."""
    from fastdm_amd.kernel.operators_set import rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    g = gen(head + rot + off)
    B, S, Hq, Hk, C = 2, 19, 6, 2, 40
    wide = off + (Hq + 2 * Hk) * head + 5
    qkv = randn(g, B, S, wide)
    positions = torch.randint(0, 5000, (S, B), generator=g, device="cuda").t()          # (strided itself)
    freqs = RotaryFrequencies(rot, device="cuda")
    q_at, k_at = slice(off, off + Hq * head), slice(off + Hq * head, off + (Hq + Hk) * head)
    (q64, qtol), (k64, ktol) = (rope64(qkv[..., a], head, freqs, positions, is_neox) for a in (q_at, k_at))
    qo, ko = rotary_positions(qkv[..., q_at], qkv[..., k_at], head, freqs, positions, is_neox=is_neox)
    assert_within(qo, q64, qtol, "q")
    assert_within(ko, k64, ktol, "k")
    mine, cache = qkv.clone(), randn(g, B, C, Hk * head)
    kept = cache.clone()
    got, into = rotary_positions(mine[..., q_at], mine[..., k_at], head, freqs, positions, is_neox=is_neox, query_out=mine[..., q_at], key_out=cache[:, 11:11 + S])
    assert got.data_ptr() == mine[..., q_at].data_ptr() and into.data_ptr() == cache[:, 11:].data_ptr()
    assert torch.equal(mine[..., q_at], qo) and torch.equal(cache[:, 11:11 + S], ko)
    assert torch.equal(mine[..., :off], qkv[..., :off]) and torch.equal(mine[..., q_at.stop:], qkv[..., q_at.stop:])
    assert torch.equal(cache[:, :11], kept[:, :11]) and torch.equal(cache[:, 11 + S:], kept[:, 11 + S:])
    alone, none = rotary_positions(qkv[..., q_at], None, head, freqs, positions, is_neox=is_neox)
    assert none is None and torch.equal(alone, qo)
    turned = qkv[:, :, q_at].transpose(0, 1).contiguous().transpose(0, 1)               # token-major storage: batch stride < token stride
    assert torch.equal(rotary_positions(turned, None, head, freqs, positions, is_neox=is_neox)[0], qo)


def test_rotary_positions_agrees_with_the_table_operator_and_keeps_relative_angles():
    """At places 0 .. S - 1 it is rotary_pos_embedding up to that operator's bf16 table and its three roundings; scores depend on distances alone."""
    from fastdm_amd.kernel.operators_set import rotary_pos_embedding, rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    g = gen(5)
    B, S, H, D = 2, 50, 4, 64
    q, k = randn(g, B, S, H * D), randn(g, B, S, H * D)
    freqs = RotaryFrequencies(D, device="cuda")
    angle = torch.arange(S, dtype=torch.float64)[:, None] * torch.tensor(freqs.theta, dtype=torch.float64)
    table = torch.cat((angle.cos(), angle.sin()), -1).to(BF16).cuda()
    for neox in (False, True):
        qo, ko = rotary_positions(q, k, D, freqs, is_neox=neox)
        q2, k2 = q.clone(), k.clone()
        rotary_pos_embedding(q2, k2, D, table, is_neox=neox)
        for a, b, x in ((qo, q2, q), (ko, k2, k)):
            # table entries, two products and the difference each round to bf16 there (at most 2^-8 of |a| and of |b| three times), and once here
            limit = 4 * HALF_STEP * 2 * x.double().abs().reshape(B, S, H, D).amax(-1, keepdim=True).expand(B, S, H, D).reshape(B, S, H * D)
            assert_within(a, b.double(), limit, "against the table")
        far = 700000
        qa, ka = rotary_positions(q, k, D, freqs, torch.arange(S, device="cuda") + far, is_neox=neox)
        near = (qo.double().view(B, S, H, D) * ko.double().view(B, S, H, D).flip(1)).sum(-1)
        away = (qa.double().view(B, S, H, D) * ka.double().view(B, S, H, D).flip(1)).sum(-1)
        # every q and k element is rounded once (2^-8): a product of two moves by 2 * 2^-8 of itself on each side
        size = (q.double().norm(dim=-1).unsqueeze(-1) * k.double().flip(1).norm(dim=-1).unsqueeze(-1))
        assert ((near - away).abs() <= 4.1 * HALF_STEP * size).all()


def test_rotary_positions_of_no_tokens():
    from fastdm_amd.kernel.operators_set import rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    freqs = RotaryFrequencies(64, device="cuda")
    q, k = rotary_positions(torch.empty(2, 0, 128, device="cuda", dtype=BF16), torch.empty(2, 0, 64, device="cuda", dtype=BF16), 64, freqs)
    assert q.shape == (2, 0, 128) and k.shape == (2, 0, 64)


# ================================================================================================ window_scaled_dot_product_attention
def window64(q, k, v, Hq, Hk, D, window, sinks, scale=None, q_lens=None, kv_lens=None):
    """In 64 bits, one sequence and kv head at a time, over the visible keys alone; and the tolerance element by element."""
    B, S, _ = q.shape
    L = k.shape[1]
    scale, window, sinks = D ** -0.5 if scale is None else scale, min(window, L + 1), min(sinks, L)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    G = Hq // Hk
    for b in range(B):
        qn = S if q_lens is None else min(max(int(q_lens[b]), 0), S)
        kn = L if kv_lens is None else min(max(int(kv_lens[b]), 0), L)
        if qn == 0 or kn == 0:
            continue
        place = (kn - qn + torch.arange(qn, device=q.device))[:, None]
        j = torch.arange(kn, device=q.device)[None]
        see = (j <= place) & ((place - j < window) | (j < sinks))
        for hk in range(Hk):
            kk, vv = k[b, :kn, hk * D:(hk + 1) * D].double(), v[b, :kn, hk * D:(hk + 1) * D].double()
            some = see.any(0)                                # what nobody sees may be anything: left out of the products
            kk, vv = kk[some], vv[some]
            sub = see[:, some]
            for g in range(G):
                at = slice((hk * G + g) * D, (hk * G + g + 1) * D)
                qq = q[b, :qn, at].double()
                s = ((qq @ kk.t()) * scale).masked_fill(~sub, -math.inf)
                any_ = sub.any(1, keepdim=True)
                p = torch.where(any_, torch.softmax(s, -1), torch.zeros_like(s))
                o, size = p @ vv, p @ vv.abs()
                # scores: D products summed in fp32, scaled and shifted (each step 2^-24 of the sum of magnitudes); 2^x to 2^-22.  A weight and the weights'
                # sum are off by that, relative; the weight is rounded to bf16, and the result once more
                delta = (D + 4) * 2.0 ** -24 * scale * ((qq.abs() @ kk.abs().t()) * sub).amax(1, keepdim=True)
                out[b, :qn, at] = o
                tol[b, :qn, at] = o.abs() * HALF_STEP + size * (HALF_STEP + 2 * delta + 2.0 ** -20) * (1 + HALF_STEP)
    return out, tol


def check_window(q, k, v, Hq, Hk, D, window, sinks, what="window", **kw):
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention
    got = window_scaled_dot_product_attention(q, k, v, Hq, Hk, D, window, sinks=sinks, **kw)
    want, tol = window64(q, k, v, Hq, Hk, D, window, sinks, **kw)
    assert_within(got, want, tol, what)
    return got


def lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,L,window,sinks", [(1, 1, 1, 0), (1, 1, 4, 3), (2, 2, 1, 0), (5, 5, 2, 1), (63, 63, 7, 0), (64, 64, 64, 4), (65, 65, 16, 2), (200, 200, 1000, 0),
                                              (130, 130, 1, 1), (257, 257, 64, 64), (300, 300, 33, 130), (129, 500, 100, 5), (1, 700, 65, 3), (3, 333, 40, 129),
                                              (8, 1025, 256, 0), (1, 4100, 4096, 4), (700, 700, 128, 10), (31, 2000, 500, 1), (513, 1025, 300, 7)])
def test_window_attention(S, L, window, sinks, D):
    g = gen(S * 7 + L + window + sinks + D)
    for B, Hq, Hk in ((1, 4, 4), (2, 8, 2), (1, 7, 1), (3, 3, 3)):
        q, k, v = randn(g, B, S, Hq * D, scale=2.0), randn(g, B, L, Hk * D), randn(g, B, L, Hk * D)
        check_window(q, k, v, Hq, Hk, D, window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,L,window,sinks", [(150, 150, 40, 3), (150, 400, 64, 70), (1, 900, 100, 2), (4, 900, 600, 1)])
def test_window_attention_of_ragged_batches(S, L, window, sinks, D):
    """Padded batches and part-filled caches, empty sequences, more queries than tokens (rows that see nothing), lengths out of range."""
    g = gen(S + L + D)
    B, Hq, Hk = 6, 6, 2
    q, k, v = randn(g, B, S, Hq * D), randn(g, B, L, Hk * D), randn(g, B, L, Hk * D)
    kv = lens(L, L // 2, 1, 0, max(1, S // 2), L + 50)
    qn = lens(S, S // 2, 1, S, S, 2 * S)
    check_window(q, k, v, Hq, Hk, D, window, sinks, kv_lens=kv)
    check_window(q, k, v, Hq, Hk, D, window, sinks, q_lens=qn)
    got = check_window(q, k, v, Hq, Hk, D, window, sinks, q_lens=qn, kv_lens=kv)
    assert (got[3] == 0).all() and (got[1, S // 2:] == 0).all()                # an empty sequence; rows past the queries
    negative = lens(-3, S, S, S, S, S)
    assert (check_window(q, k, v, Hq, Hk, D, window, sinks, q_lens=negative)[0] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_on_slices_of_a_projection_and_a_cache(D):
    """q from a fused projection; k and v from caches with other orders of the axes, and one sequence's cache shared by the whole batch."""
    g = gen(D)
    B, S, L, Hq, Hk = 3, 70, 260, 4, 2
    qkv = randn(g, B, S, (Hq + 2 * Hk) * D + 8)
    q = qkv[..., 8:8 + Hq * D]
    cache = randn(g, L + 40, B, 2, Hk * D)                                     # token-major, k and v side by side
    k, v = cache[10:10 + L, :, 0].transpose(0, 1), cache[10:10 + L, :, 1].transpose(0, 1)
    plain = check_window(q.contiguous(), k.contiguous(), v.contiguous(), Hq, Hk, D, 50, 5)
    assert torch.equal(check_window(q, k, v, Hq, Hk, D, 50, 5), plain)
    shared = k[:1].expand(B, L, Hk * D)
    assert torch.equal(check_window(q, shared, v, Hq, Hk, D, 50, 5), check_window(q, shared.contiguous(), v, Hq, Hk, D, 50, 5))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,L", [(1, 400), (5, 400), (90, 400), (300, 300)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_window_attention_keeps_what_is_not_seen_out(S, L, bad, D):
    """Keys past the lengths, keys in front of every window and behind the sinks hold anything; a value some rows see reaches those rows alone."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(S + D)
    B, Hq, Hk, window, sinks = 2, 6, 2, 37, 3
    q, k, v = randn(g, B, S, Hq * D), randn(g, B, L, Hk * D), randn(g, B, L, Hk * D)
    kv = lens(L - 30, L)
    qn = lens(min(S, L - 30), S)
    clean = check_window(q, k, v, Hq, Hk, D, window, sinks, q_lens=qn, kv_lens=kv)
    k2, v2 = k.clone(), v.clone()
    k2[0, L - 30:], v2[0, L - 30:] = bad, bad
    for b, (n, t) in enumerate(((L - 30, min(S, L - 30)), (L, S))):
        front = max(sinks, n - t - window + 1)
        k2[b, sinks:front], v2[b, sinks:front] = bad, bad
    assert torch.equal(attend(q, k2, v2, Hq, Hk, D, window, sinks=sinks, q_lens=qn, kv_lens=kv), clean)
    if S > 1:
        # a bad value inside: key j of sequence 1, seen by the rows at places j .. j + window - 1
        j = L - S // 2 - 1
        v3 = v.clone()
        v3[1, j] = bad
        got = attend(q, k, v3, Hq, Hk, D, window, sinks=sinks, q_lens=qn, kv_lens=kv)
        place = torch.arange(L - S, L, device="cuda")
        sees = (place >= j) & (place < j + window)
        assert torch.equal(got[1, ~sees], clean[1, ~sees]) and torch.equal(got[0], clean[0])
        assert not torch.isfinite(got[1, sees]).any()
        k3 = k.clone()
        k3[1, j] = bad
        got = attend(q, k3, v, Hq, Hk, D, window, sinks=sinks, q_lens=qn, kv_lens=kv)
        assert torch.equal(got[1, ~sees], clean[1, ~sees])


def test_window_attention_scores_of_every_size():
    """Large, small and equal scores: the running maximum moves, stays, and starts far below."""
    g = gen(9)
    D, S = 64, 200
    for scale, offset in ((50.0, 0.0), (1e-6, 0.0), (1.0, 0.0), (1.0, 1e4), (1.0, -1e4)):
        q, k, v = randn(g, 1, S, 2 * D), randn(g, 1, S, 2 * D), randn(g, 1, S, 2 * D)
        if offset:
            q[..., 0], k[..., 0] = 100.0, offset
            q[..., D], k[..., D] = 100.0, offset
        check_window(q, k, v, 2, 2, D, 64, 4, scale=scale * D ** -0.5)
    one = torch.zeros(1, S, 2 * D, device="cuda", dtype=BF16)
    check_window(one, one, randn(g, 1, S, 2 * D), 2, 2, D, 64, 4)


@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_with_an_open_window_is_causal_attention(D):
    from fastdm_amd.kernel.operators_set import scaled_dot_product_attention
    g = gen(D + 1)
    S, H = 333, 3
    q, k, v = randn(g, 1, S, H * D), randn(g, 1, S, H * D), randn(g, 1, S, H * D)
    got = check_window(q, k, v, H, H, D, 1 << 40, 0)
    want, tol = window64(q, k, v, H, H, D, S, 0)
    assert_within(scaled_dot_product_attention(q, k, v, H, H, D, is_causal=True), want, tol, "causal")
    assert_within(got, want, tol, "open window")


def test_window_attention_parts_agree_with_whole_lists():
    """The same token attended alone (its tiles in parts, merged) and as the last row of a long batch of tokens (whole lists)."""
    g = gen(11)
    D, Hq, Hk, L = 128, 8, 2, 5000
    q, k, v = randn(g, 1, L, Hq * D), randn(g, 1, L, Hk * D), randn(g, 1, L, Hk * D)
    whole = check_window(q[:, -600:], k, v, Hq, Hk, D, 3000, 9)
    for n in (1, 2, 8, 9, 40):
        part = check_window(q[:, -n:].contiguous(), k, v, Hq, Hk, D, 3000, 9)
        want, tol = window64(q[:, -n:], k, v, Hq, Hk, D, 3000, 9)
        assert ((part.double() - whole[:, -n:].double()).abs() <= 2 * tol).all()


def test_window_attention_repeats_bit_for_bit_on_streams_and_in_graphs():
    """Two captured graphs, replayed in turn with eager calls between, and calls on two streams at once: each its own workspace."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(12)
    D, Hq, Hk, L = 128, 8, 2, 6000
    sets = [(randn(g, 2, 1, Hq * D), randn(g, 2, L, Hk * D), randn(g, 2, L, Hk * D)) for _ in range(2)]
    kv = [lens(L, L - 777), lens(L - 1, 4000)]
    want = [attend(*s, Hq, Hk, D, 4000, sinks=4, kv_lens=n) for s, n in zip(sets, kv)]
    assert not torch.equal(want[0], want[1])
    graphs, outs = [], []
    for s, n in zip(sets, kv):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attend(*s, Hq, Hk, D, 4000, sinks=4, kv_lens=n))
        graphs.append(graph)
    for _ in range(4):
        for i in (0, 1):
            outs[i].zero_()
            graphs[i].replay()
            assert torch.equal(attend(*sets[1 - i], Hq, Hk, D, 4000, sinks=4, kv_lens=kv[1 - i]), want[1 - i])
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = attend(*sets[i], Hq, Hk, D, 4000, sinks=4, kv_lens=kv[i])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_window_attention_of_nothing():
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    e = lambda *s: torch.empty(*s, device="cuda", dtype=BF16)  # noqa: E731
    assert attend(e(0, 4, 128), e(0, 4, 128), e(0, 4, 128), 2, 2, 64, 4).shape == (0, 4, 128)
    assert attend(e(2, 0, 128), e(2, 4, 128), e(2, 4, 128), 2, 2, 64, 4).shape == (2, 0, 128)
    q = torch.ones(2, 3, 128, device="cuda", dtype=BF16)
    assert (attend(q, e(2, 0, 128), e(2, 0, 128), 2, 2, 64, 4) == 0).all()     # no keys: rows that see nothing


def test_window_attention_behind_offsets_over_32_bits():
    """A cache of more than 2^32 elements: the last sequence's keys lie past every 32-bit offset."""
    D, Hk, Hq, B, L = 128, 8, 8, 5, 1 << 20
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    k = torch.zeros(B, L, Hk * D, device="cuda", dtype=BF16)
    v = torch.zeros(B, L, Hk * D, device="cuda", dtype=BF16)
    assert k.numel() > 1 << 32
    g = gen(13)
    q = randn(g, B, 1, Hq * D)
    k[:, -600:], v[:, -600:] = randn(g, B, 600, Hk * D), randn(g, B, 600, Hk * D)
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    got = attend(q, k, v, Hq, Hk, D, 500)
    want, tol = window64(q, k[:, -600:], v[:, -600:], Hq, Hk, D, 500, 0)
    assert_within(got, want, tol, "far keys")


@pytest.mark.parametrize("bad", [None, float("nan")])
@pytest.mark.parametrize("B,S,L,Hq,Hk,D,window,sinks", [(8, 300, 300, 12, 12, 64, 100, 5), (8, 300, 420, 12, 12, 128, 100, 70), (3, 411, 411, 56, 8, 128, 64, 1),
                                                        (5, 260, 2600, 4, 2, 128, 2100, 130), (1, 515, 3000, 16, 4, 128, 2500, 0), (9, 130, 130, 48, 16, 64, 200, 0)])
def test_window_attention_of_many_blocks_and_of_long_lists(B, S, L, Hq, Hk, D, window, sinks, bad):
    """Row blocks that fill the chip, and long lists of few blocks: ragged, with neighbours that are not numbers."""
    g = gen(B * S + L + D)
    q, k, v = randn(g, B, S, Hq * D, scale=1.5), randn(g, B, L, Hk * D), randn(g, B, L, Hk * D)
    qn = lens(*[S - 17 * b for b in range(B)])
    kv = lens(*[L - 29 * b for b in range(B)])
    clean = check_window(q, k, v, Hq, Hk, D, window, sinks, q_lens=qn, kv_lens=kv)
    if bad is None:
        check_window(q, k, v, Hq, Hk, D, window, sinks)
        return
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    j = L - S // 2
    sees = []
    for b in range(B):
        kv_len, q_len = L - 29 * b, S - 17 * b
        k[b, kv_len:], v[b, kv_len:] = bad, bad
        front = max(sinks, kv_len - q_len - window + 1)
        k[b, sinks:front], v[b, sinks:front] = bad, bad
        row = torch.arange(S, device="cuda")
        place = kv_len - q_len + row
        sees.append((row < q_len) & (place >= j) & ((place < j + window) | (j < sinks)) if j < kv_len else torch.zeros(S, dtype=torch.bool, device="cuda"))
        if j < kv_len:
            v[b, j, 5::D] = bad                       # one element of every kv head's value
    got = attend(q, k, v, Hq, Hk, D, window, sinks=sinks, q_lens=qn, kv_lens=kv)
    hit = torch.stack(sees)[:, :, None] & (torch.arange(Hq * D, device="cuda") % D == 5)
    assert hit.any() and torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


def test_window_attention_takes_any_stride_of_an_axis_of_one():
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(21)
    q, k, v = randn(g, 1, 1, 256), randn(g, 1, 50, 128), randn(g, 1, 50, 128)
    want = check_window(q, k, v, 4, 2, 64, 1 << 70, 1 << 70)
    odd = [torch.as_strided(t, t.shape, (t.stride(0) + 3, t.stride(1) if t.shape[1] > 1 else 5, 1)) for t in (q, k, v)]
    assert torch.equal(attend(*odd, 4, 2, 64, 50, sinks=3), want)
    one = attend(q, torch.as_strided(k, (1, 1, 128), (7, 9, 1)), torch.as_strided(v, (1, 1, 128), (7, 9, 1)), 4, 2, 64, 1)
    assert torch.equal(one.view(2, 2, 64), v[0, 0].view(2, 1, 64).expand(2, 2, 64))


# ================================================================================================ together
class DecoderAttention:
    """The attention half of a decoder layer as a program that serves runs it: the residual's addition and norm into e4m3, the fused W8A8 projection, rotary
    positions of q and of k straight into the cache, attention over the cache."""

    def __init__(self, seed, width, Hq, Hk, D, window, sinks, batch, room):
        from fastdm_amd.kernel.operators_set import quantize_to_fp8
        from fastdm_amd.layer.embeddings import RotaryFrequencies
        g = gen(seed)
        self.Hq, self.Hk, self.D, self.window, self.sinks = Hq, Hk, D, window, sinks
        self.weight = (1 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(BF16)
        self.proj, self.proj_scale = quantize_to_fp8(randn(g, (Hq + 2 * Hk) * D, width, scale=width ** -0.5))
        self.freqs = RotaryFrequencies(D, base=500000.0, scaling="yarn", factor=4.0, original_length=64, device="cuda")
        self.k, self.v = (torch.full((batch, room, Hk * D), float("nan"), device="cuda", dtype=BF16) for _ in range(2))

    def __call__(self, x, residual, at, q_lens=None, kv_lens=None):
        """Tokens at .. at + S - 1 of every sequence; returns (attention's output, the new residual, q)."""
        from fastdm_amd.kernel.fused import add_rms_norm
        from fastdm_amd.kernel.operators_set import fp8_matmul, rotary_positions, window_scaled_dot_product_attention
        B, S, width = x.shape
        qw, kw = self.Hq * self.D, self.Hk * self.D
        _, z, h = add_rms_norm(x.view(B * S, width), residual.view(B * S, width), self.weight, 1e-6, quant=FP8)
        qkv = fp8_matmul(z.q, self.proj.t(), z.scale, self.proj_scale, BF16).view(B, S, qw + 2 * kw)
        positions = torch.arange(at, at + S, device="cuda")
        q, _ = rotary_positions(qkv[..., :qw], qkv[..., qw:qw + kw], self.D, self.freqs, positions, is_neox=True, key_out=self.k[:, at:at + S])
        self.v[:, at:at + S] = qkv[..., qw + kw:]
        o = window_scaled_dot_product_attention(q, self.k[:, :at + S], self.v[:, :at + S], self.Hq, self.Hk, self.D, self.window, sinks=self.sinks,
                                                q_lens=q_lens, kv_lens=kv_lens)
        return o, h.view(B, S, width), q


@pytest.mark.parametrize("D", [64, 128])
def test_decoder_attention_prompt_then_single_tokens(D):
    """A prompt in one call, in chunks, and token by token give the same rows: the row operators bit for bit, attention within its tolerance; the
    cache is NaN where nothing was written yet."""
    B, S, width, Hq, Hk, window, sinks = 2, 150, 512, 8, 2, 48, 3
    g = gen(31)
    x, residual = randn(g, B, S, width), randn(g, B, S, width, scale=3.0)
    whole = DecoderAttention(5, width, Hq, Hk, D, window, sinks, B, S)
    o, h, q = whole(x, residual, 0)
    want, tol = window64(q, whole.k, whole.v, Hq, Hk, D, window, sinks)
    assert_within(o, want, tol, "prompt")
    for sizes in ([100, 33, 17], [140] + [1] * 10):
        parts, at = DecoderAttention(5, width, Hq, Hk, D, window, sinks, B, S), 0
        for n in sizes:
            got, hn, qn = parts(x[:, at:at + n].contiguous(), residual[:, at:at + n].contiguous(), at)
            assert torch.equal(hn, h[:, at:at + n])
            # the projection's kernel goes by its number of rows: its sums may be taken in another order, so its rows are compared through attention alone
            w, t = window64(qn, parts.k[:, :at + n], parts.v[:, :at + n], Hq, Hk, D, window, sinks)
            assert_within(got, w, t, f"{n} tokens at {at}")
            at += n
        assert torch.isfinite(parts.k).all() and torch.isfinite(parts.v).all()


def test_decoder_attention_step_in_a_graph():
    """One token's step captured once and replayed for growing sequences (lengths and positions are device tensors), eager work and waits between."""
    from fastdm_amd.kernel.fused import add_rms_norm
    from fastdm_amd.kernel.operators_set import rotary_positions, window_scaled_dot_product_attention
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    B, Hq, Hk, D, room, width = 3, 8, 2, 64, 900, 512
    g = gen(41)
    k, v = randn(g, B, room, Hk * D), randn(g, B, room, Hk * D)
    x, residual = randn(g, B, width), randn(g, B, width)
    weight = randn(g, width)
    freqs = RotaryFrequencies(D, device="cuda")
    kv = lens(600, 1, 300)
    positions = torch.zeros(B, 1, dtype=torch.int64, device="cuda")

    def step():
        y, _, h = add_rms_norm(x, residual, weight, 1e-6)
        q, _ = rotary_positions(y.view(B, 1, width), None, D, freqs, positions)
        return h, q, window_scaled_dot_product_attention(q, k, v, Hq, Hk, D, 512, sinks=2, kv_lens=kv)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(randn(g, B, width))
        kv.copy_(lens(600 + 7 * i, 1 + 250 * i, room - i))
        positions.copy_(kv.long()[:, None] - 1)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)
        want, tol = window64(out[1], k, v, Hq, Hk, D, 512, 2, kv_lens=kv)
        assert_within(out[2], want, tol, "replayed")


def test_calls_that_would_lose_a_gradient_and_mixed_devices_are_refused():
    from fastdm_amd.kernel.fused import add_rms_norm
    from fastdm_amd.kernel.operators_set import rotary_positions, window_scaled_dot_product_attention
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    x = randn(gen(51), 4, 64)
    w = torch.ones(64, device="cuda", dtype=BF16)
    leaf = x.clone().requires_grad_()
    freqs = RotaryFrequencies(64, device="cuda")
    with pytest.raises(RuntimeError, match="forward only"):
        add_rms_norm(leaf, None, w, 1e-6)
    with pytest.raises(RuntimeError, match="forward only"):
        rotary_positions(leaf[None], None, 64, freqs)
    with pytest.raises(RuntimeError, match="forward only"):
        window_scaled_dot_product_attention(x[None], leaf[None], x[None], 1, 1, 64, 4)
    with torch.no_grad():
        add_rms_norm(leaf, None, w, 1e-6)
    with pytest.raises(RuntimeError, match="GPU"):
        add_rms_norm(x, x.cpu(), w, 1e-6)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_positions(x[None], None, 64, RotaryFrequencies(64))
    with pytest.raises(RuntimeError, match="GPU"):
        window_scaled_dot_product_attention(x[None], x[None], x[None], 1, 1, 64, 4, kv_lens=torch.tensor([4], dtype=torch.int32))


@pytest.mark.parametrize("what", ["dtype", "shape", "heads", "head_dim", "window", "sinks", "scale", "lens dtype", "lens shape", "inner stride", "alignment", "batch"])
def test_window_attention_refusals(what):
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    q, k = randn(gen(1), 2, 5, 256), randn(gen(2), 2, 9, 128)
    a = dict(q=q, k=k, v=k, hq=4, hk=2, D=64, window=4, kw={})
    change = {"dtype": dict(q=q.half()), "shape": dict(v=k[:, :8]), "heads": dict(hq=3, q=q[..., :192]), "head_dim": dict(D=32, hq=8, hk=4), "window": dict(window=0),
              "sinks": dict(kw=dict(sinks=-1)), "scale": dict(kw=dict(scale=0.0)), "lens dtype": dict(kw=dict(kv_lens=torch.ones(2, dtype=torch.int64, device="cuda"))),
              "lens shape": dict(kw=dict(q_lens=lens(1, 2, 3))), "inner stride": dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
              "alignment": dict(q=torch.cat((q, q), -1)[..., 4:260]), "batch": dict(k=k[:1], v=k[:1])}[what]
    a.update(change)
    with pytest.raises((AssertionError, RuntimeError)):
        attend(a["q"], a["k"], a["v"], a["hq"], a["hk"], a["D"], a["window"], **a["kw"])


@pytest.mark.parametrize("what", ["dtype", "width", "residual", "quant", "out without residual", "rows", "inner stride"])
def test_add_rms_norm_refusals(what):
    from fastdm_amd.kernel.fused import add_rms_norm
    x, w = randn(gen(1), 6, 64), torch.ones(64, device="cuda", dtype=BF16)
    call = {"dtype": lambda: add_rms_norm(x.float(), None, w, 1e-6), "width": lambda: add_rms_norm(x, None, w[:32], 1e-6), "residual": lambda: add_rms_norm(x, x[:3], w, 1e-6),
            "quant": lambda: add_rms_norm(x, None, w, 1e-6, quant=torch.uint8), "out without residual": lambda: add_rms_norm(x, None, w, 1e-6, residual_out=x),
            "rows": lambda: add_rms_norm(x[:1].expand(6, 64), None, w, 1e-6), "inner stride": lambda: add_rms_norm(randn(gen(1), 64, 6).t(), None, w, 1e-6)}[what]
    with pytest.raises((AssertionError, RuntimeError)):
        call()


@pytest.mark.parametrize("what", ["rot", "shape", "head", "positions dtype", "positions shape", "out shape", "out overlaps", "in place strides", "key out without key"])
def test_rotary_positions_refusals(what):
    from fastdm_amd.kernel.operators_set import rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    f = RotaryFrequencies(64, device="cuda")
    q = randn(gen(1), 2, 6, 128)
    call = {"rot": lambda: rotary_positions(q, None, 32, f), "shape": lambda: rotary_positions(q, q[:, :5], 64, f), "head": lambda: rotary_positions(q, None, 96, f),
            "positions dtype": lambda: rotary_positions(q, None, 64, f, torch.zeros(6, device="cuda")), "positions shape": lambda: rotary_positions(q, None, 64, f, torch.zeros(5, dtype=torch.int64, device="cuda")),
            "out shape": lambda: rotary_positions(q, None, 64, f, query_out=q[:, :5]), "out overlaps": lambda: rotary_positions(q, None, 64, f, query_out=q[:1].expand(2, 6, 128)),
            "in place strides": lambda: rotary_positions(q, None, 64, f, query_out=torch.as_strided(q, (2, 6, 128), (128, 256, 1))),
            "key out without key": lambda: rotary_positions(q, None, 64, f, key_out=q)}[what]
    with pytest.raises((AssertionError, RuntimeError)):
        call()


@pytest.mark.parametrize("what", ["next rows", "next columns", "other strides", "query_out on key", "key_out on query", "key_out on query_out", "query_out a token on"])
def test_outputs_across_inputs_are_refused(what):
    from fastdm_amd.kernel.fused import add_rms_norm
    from fastdm_amd.kernel.operators_set import rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    m, w, f = randn(gen(1), 8, 128), torch.ones(64, device="cuda", dtype=BF16), RotaryFrequencies(64, device="cuda")
    kept = m.clone()
    x, r, t = m[:4, :64], randn(gen(2), 4, 64), m[None]
    q, k, o = t[:, :6, :64], t[:, :6, 64:], randn(gen(3), 1, 6, 64)
    call = {"next rows": lambda: add_rms_norm(x, r, w, 1e-6, residual_out=m[1:5, :64]), "next columns": lambda: add_rms_norm(r, x, w, 1e-6, residual_out=m[:4, 32:96]),
            "other strides": lambda: add_rms_norm(x, r, w, 1e-6, residual_out=m.view(16, 64)[:4]),
            "query_out on key": lambda: rotary_positions(q, k, 64, f, query_out=k), "key_out on query": lambda: rotary_positions(q, k, 64, f, query_out=o, key_out=q),
            "key_out on query_out": lambda: rotary_positions(q, k, 64, f, query_out=o, key_out=o), "query_out a token on": lambda: rotary_positions(q, k, 64, f, query_out=t[:, 1:7, :64])}[what]
    with pytest.raises(AssertionError):
        call()
    assert torch.equal(m, kept)
