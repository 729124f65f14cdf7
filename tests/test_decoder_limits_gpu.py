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
