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
@pytest.mark.parametrize("head,rot", [(128, 128), (64, 32), (64, 64), (80, 20), (96, 24), (256, 256), (256, 64), (10, 6), (7, 2), (128, 12)])
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
