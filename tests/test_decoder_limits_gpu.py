"""GPU: the decoder-side operators on sizes past what one launch carries (2^32 threads), and at the edges of what rows may hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(BF16)


def need(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB")


# ================================================================================================ more threads than a launch holds
@pytest.mark.parametrize("quant", [None, FP8, torch.int8])
def test_add_rms_norm_of_more_rows_than_a_launch_holds(quant):
    """2^26 rows and more, 64 threads each: every copy of a block of rows gives what the block alone gives, bit for bit."""
    from fastdm_amd.kernel.fused import add_rms_norm
    need(24)
    rows, copies, width = 16411, 4096, 8
    assert rows * copies * 64 > 1 << 32
    g = gen(1)
    x, r, w = randn(g, rows, width), randn(g, rows, width), randn(g, width)
    out, z, h = add_rms_norm(x, r, w, 1e-6, quant=quant)
    many = [t.expand(copies, rows, width).reshape(-1, width) for t in (x, r)]
    out2, z2, h2 = add_rms_norm(*many, w, 1e-6, quant=quant)
    pairs = [(h, h2)] + ([(out, out2)] if quant is None else [(z.q.view(torch.uint8), z2.q.view(torch.uint8)), (z.scale, z2.scale)])
    if quant == torch.int8:
        pairs.append((z.azp, z2.azp))
    for one, all_ in pairs:
        assert bool((all_.view(copies, rows, -1) == one).all())


@pytest.mark.parametrize("is_neox", [False, True])
def test_rotary_positions_of_more_tokens_than_a_launch_holds(is_neox):
    """2^28 tokens of one pair and more, 16 to a block of 256 threads."""
    from fastdm_amd.kernel.operators_set import rotary_positions
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    need(16)
    B, S = 16411, 16384
    assert B * S // 16 * 256 > 1 << 32
    g = gen(2)
    q, k = randn(g, 1, S, 2), randn(g, 1, S, 2)
    freqs = RotaryFrequencies(2, device="cuda")
    qo, ko = rotary_positions(q, k, 2, freqs, is_neox=is_neox)
    many = [t.expand(B, S, 2).contiguous() for t in (q, k)]
    for one, all_ in zip((qo, ko), rotary_positions(*many, 2, freqs, is_neox=is_neox)):
        assert bool((all_ == one).all())


def test_window_attention_of_more_blocks_than_a_launch_holds():
    """2^26 pairs of sequence and head and more, a wave each, that see one key: its value."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention
    need(64)
    rows, copies, H, D = 4093, 4096, 5, 64
    B = rows * copies
    assert B * H * 64 > 1 << 32
    g = gen(3)
    q, k, v = (randn(g, rows, 1, H * D) for _ in range(3))
    many = v.view(1, rows, H * D).expand(copies, rows, H * D).reshape(B, 1, H * D)
    got = window_scaled_dot_product_attention(q[:1].expand(B, 1, H * D), k[:1].expand(B, 1, H * D), many, H, H, D, 4)
    # one key: the weight is 2^(s - s') with s' = s up to its last bit, bf16(weight) = 1; the division by the unrounded weight is off by 2^-22 of the value, a
    # bf16 number: it rounds back to it
    assert bool((got.view(copies, rows, H * D) == v.view(1, rows, H * D)).all())


# ================================================================================================ rows by themselves
FORMS = [(2, 9, 700, 6, 2, 64, 300, 3), (2, 1, 900, 8, 1, 128, 500, 2), (3, 90, 400, 8, 2, 64, 200, 5), (2, 100, 500, 6, 2, 128, 150, 70),
         (8, 300, 420, 12, 12, 64, 200, 5), (3, 411, 411, 56, 8, 128, 128, 1), (1, 515, 3000, 16, 4, 128, 2500, 0)]      # each form, G = 1 and more


@pytest.mark.parametrize("B,S,L,Hq,Hk,D,window,sinks", FORMS)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 1e30, -1e30, "large"])
def test_window_attention_rows_past_the_queries_change_no_bit(B, S, L, Hq, Hk, D, window, sinks, fill):
    """What a padded batch holds past q_lens: the queries in front of it, which share waves with it, keep every bit."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    if S == 1:
        pytest.skip("one query: nothing behind it")
    g = gen(S + L + D)
    q, k, v = randn(g, B, S, Hq * D, scale=1.5), randn(g, B, L, Hk * D), randn(g, B, L, Hk * D)
    lengths = [max(1, S - 3 - 7 * b) for b in range(B)]
    q_lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    other = q.clone()
    for b, n in enumerate(lengths):
        q[b, n:] = 0
        other[b, n:] = randn(g, S - n, Hq * D, scale=500.0) if fill == "large" else fill
    want = attend(q, k, v, Hq, Hk, D, window, sinks=sinks, q_lens=q_lens)
    assert torch.isfinite(want).all() and torch.equal(attend(other, k, v, Hq, Hk, D, window, sinks=sinks, q_lens=q_lens), want)


@pytest.mark.parametrize("B,S,L,Hq,Hk,D,window,sinks", FORMS)
def test_window_attention_rows_do_not_go_by_their_neighbours(B, S, L, Hq, Hk, D, window, sinks):
    """Other queries of the same wave that meet far larger scores, and a key that only some rows see with an infinity in it: the other rows keep every bit."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(S * L + D)
    q, k, v = randn(g, B, S, Hq * D, scale=1.5), randn(g, B, L, Hk * D), randn(g, B, L, Hk * D)
    want = attend(q, k, v, Hq, Hk, D, window, sinks=sinks)
    loud = q.view(B, S, Hq, D).clone()
    row = torch.arange(S, device="cuda")[:, None] * Hq + torch.arange(Hq, device="cuda")[None]
    loud[:, row % 3 == 1] *= 60.0
    got = attend(loud.view_as(q), k, v, Hq, Hk, D, window, sinks=sinks)
    quiet = (row % 3 != 1)[None, :, :, None].expand(B, S, Hq, D)
    assert torch.equal(got.view(B, S, Hq, D)[quiet], want.view(B, S, Hq, D)[quiet])
    if S > 1:
        j = L - S // 2 - 1
        for bad in (float("inf"), -float("inf")):
            k2 = k.clone()
            k2[:, j, ::D] = bad                  # one element of every kv head's key
            got = attend(q, k2, v, Hq, Hk, D, window, sinks=sinks)
            place = torch.arange(L - S, L, device="cuda")
            sees = (place >= j) & ((place < j + window) | (j < sinks))
            assert not sees.all() and torch.equal(got[:, ~sees], want[:, ~sees])


# ================================================================================================ rows that are not finite
@pytest.mark.parametrize("width", [8, 500, 1003, 5120, 8192, 40000])
@pytest.mark.parametrize("quant", [None, FP8, torch.int8])
def test_add_rms_norm_of_what_is_not_finite_at_any_weight(width, quant):
    """A NaN or an infinity at a channel whose weight is 0, and a NaN weight: NaN where the formula gives NaN, a NaN scale for such 8-bit rows; others as ever."""
    from fastdm_amd.kernel.fused import add_rms_norm
    g = gen(width)
    nan, inf = float("nan"), float("inf")
    x, residual = randn(g, 9, width), randn(g, 9, width)
    weight = (1 + 0.3 * torch.randn(width, generator=g, device="cuda")).to(BF16)
    at = width - 1 if width % 8 else width // 2 + 3
    weight[at] = 0
    finite = add_rms_norm(x, residual, weight, 1e-6, quant=quant)
    for row, value in ((1, nan), (3, inf), (5, -inf)):
        x[row, at] = value
    residual[7, at], x[7, at] = inf, -inf                      # their sum is NaN
    bad = torch.tensor([1, 3, 5, 7], device="cuda")
    good = torch.tensor([0, 2, 4, 6, 8], device="cuda")
    out, z, h = add_rms_norm(x, residual, weight, 1e-6, quant=quant)
    assert torch.equal(h[good], finite[2][good])
    if quant is None:
        assert torch.equal(out[good], finite[0][good]) and torch.isnan(out[bad, at]).all() and torch.isnan(out[[1, 7]]).all()
        beside = torch.arange(width, device="cuda") != at
        assert (out[[3, 5]][:, beside] == 0).all()
    else:
        assert torch.isnan(z.scale[bad]).all() and torch.equal(z.scale[good], finite[1].scale[good])
        assert torch.equal(z.q.view(torch.uint8)[good], finite[1].q.view(torch.uint8)[good])
        if quant == FP8:
            assert torch.isnan(z.q[bad].float()).all()
    weight[at] = nan
    out, z, _ = add_rms_norm(randn(g, 3, width), None, weight, 1e-6, quant=quant)
    if quant is None:
        assert torch.isnan(out[:, at]).all() and torch.isfinite(out[:, torch.arange(width, device="cuda") != at]).all()
    else:
        assert torch.isnan(z.scale).all()


def test_tangents_are_refused_on_the_gpu():
    import torch.autograd.forward_ad as forward_ad
    from fastdm_amd.kernel.fused import add_rms_norm
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    x, w = randn(gen(5), 4, 64), randn(gen(6), 64)
    want = add_rms_norm(x, None, w, 1e-6)[0]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="tangent"):
            add_rms_norm(dual, None, w, 1e-6)
        with pytest.raises(RuntimeError, match="tangent"):
            attend(x[None], dual[None], x[None], 1, 1, 64, 4)
        assert torch.equal(add_rms_norm(x, None, w, 1e-6)[0], want)
    for transform in (lambda: torch.func.jvp(lambda t: add_rms_norm(t, None, w, 1e-6)[0], (x,), (x,)),
                      lambda: torch.func.grad(lambda t: add_rms_norm(t, None, w, 1e-6)[0].float().sum())(x)):
        with pytest.raises(RuntimeError):
            transform()


# ================================================================================================ scores of every size
@pytest.mark.parametrize("B,S,L,Hq,Hk,D,window,sinks", FORMS)
@pytest.mark.parametrize("shape", ["above", "below", "climbing", "falling", "one key above"])
def test_window_attention_of_scores_with_a_large_common_part(B, S, L, Hq, Hk, D, window, sinks, shape):
    """Scores of up to 2^20 that are exact in fp32: all of them on a grid of 1/8 (queries on 1/2, keys on 1/4), so every sum of products is a whole number
    of eighths under 2^21, and what is common to a row's scores cancels in its softmax without loss.

    Then a weight is off by: the scale's rounding and the exponent's, 2^-23 of an exponent of at most 40 (smaller weights do not count), 2^x itself
    (2^-22), the sums over keys in fp32 (under 300 steps of 2^-24 for rows and products together): under 2^-15; the weight is rounded to bf16, and the
    result once more (2^-8 each)."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(S + L + Hq + D)
    q = torch.randint(-4, 5, (B, S, Hq, D), generator=g, device="cuda").double() / 2
    k = torch.randint(-8, 9, (B, L, Hk, D), generator=g, device="cuda").double() / 4
    v = randn(g, B, L, Hk, D)
    q[..., 0] = 128.0
    key = torch.arange(L, device="cuda")
    common = {"above": torch.full_like(key, 8192), "below": torch.full_like(key, -8192), "climbing": 512 * (16 * key // L), "falling": -512 * (16 * key // L),
              "one key above": torch.where(key % 97 == 50, 16, 0)}[shape]
    k[..., 0] = common.double()[None, :, None]
    assert torch.equal(q.to(BF16).double(), q) and torch.equal(k.to(BF16).double(), k)
    scale = 2.0 ** -4
    got = attend(q.to(BF16).view(B, S, Hq * D), k.to(BF16).view(B, L, Hk * D), v.view(B, L, Hk * D), Hq, Hk, D, window, sinks=sinks, scale=scale).view(B, S, Hq, D).double()
    place = torch.arange(L - S, L, device="cuda")[:, None]
    hidden = ~((key <= place) & ((place - key < window) | (key < sinks)))
    for b in range(B):
        for head in range(Hq):
            kk, vv = k[b, :, head // (Hq // Hk)], v[b, :, head // (Hq // Hk)].double()
            p = torch.softmax((q[b, :, head] @ kk.t() * scale).masked_fill(hidden, float("-inf")), -1)
            want, size = p @ vv, p @ vv.abs()
            tol = want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -15) * (1 + 2.0 ** -8)
            assert (tol < 0.01 * size + 1e-30).all()                     # (says something)
            worst = ((got[b, :, head] - want).abs() - tol).max().item()
            assert worst <= 0, f"{shape}: sequence {b}, head {head}: beyond by {worst:.3g}"


@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_of_rows_whose_scores_are_all_minus_infinity(D):
    """They have no softmax: zeros, as where a row sees nothing; one finite score beside them, and the row is that key's value."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(D)
    S, H = 90, 2
    q, k, v = randn(g, 1, S, H * D).abs() + 1, randn(g, 1, S, H * D), randn(g, 1, S, H * D)
    k[:, 10:60] = float("-inf")
    got = attend(q, k, v, H, H, D, 8)[0]
    place = torch.arange(S, device="cuda")
    none = (place >= 17) & (place < 60)
    assert (got[none] == 0).all() and torch.isfinite(got).all()
    assert torch.equal(got[16], v[0, 9]) and torch.equal(got[60], v[0, 60])


@pytest.mark.parametrize("B,S,L,Hq,Hk,D,window,sinks", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
def test_window_attention_of_scores_up_to_the_largest(B, S, L, Hq, Hk, D, window, sinks, sign):
    """Scores between 2^27 and 2^28, 2^20 and more apart in any 64 keys in a row: the largest one's key alone counts, and its value comes out.  Its weight is
    2^r, r what the maximum's rounding leaves (at most 16 at 2^28 * log2 e): no bf16 number, so it is rounded once in the product (2^-8) and not in the sum that
    the product is divided by; the result is rounded once more (2^-8), and the fp32 steps between are under 2^-20."""
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention as attend
    g = gen(D + L)
    q = torch.zeros(B, S, Hq, D, device="cuda")
    k = torch.zeros(B, L, Hk, D, device="cuda")
    v = randn(g, B, L, Hk, D)
    key = torch.arange(L, device="cuda")
    steps = (key * 37) % 127
    q[..., 0], k[..., 0] = 2.0 ** 14, sign * 2.0 ** 13 * (1 + steps / 128)[None, :, None]
    assert torch.equal(k.to(BF16).float(), k)
    got = attend(q.to(BF16).view(B, S, Hq * D), k.to(BF16).view(B, L, Hk * D), v.view(B, L, Hk * D), Hq, Hk, D, 64, scale=1.0).view(B, S, Hq, D)
    place = torch.arange(L - S, L, device="cuda")[:, None]
    seen = (key <= place) & (place - key < 64)
    best = (sign * steps).expand(S, L).masked_fill(~seen, -1000).argmax(1)
    want = v[:, best].repeat_interleave(Hq // Hk, 2).double()
    assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -15)).all()
