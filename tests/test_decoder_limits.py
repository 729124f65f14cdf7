"""CPU: the decoder-side operators at and past the sizes they can take."""
import os
import shutil
import subprocess

import pytest

from fastdm_amd import _native as N

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastdm_amd", "csrc")


def test_huge_grids_go_in_pieces_that_a_launch_can_hold(tmp_path):
    """launch_pieces: under 2^32 threads each, the blocks in order and each once, first blocks multiples of 8; ends with the first failure."""
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("needs a C++ compiler")
    source = tmp_path / "pieces.cpp"
    source.write_text("""
#include "launch.h"
#include <cstdio>
#include <initializer_list>
int main() {
  const int64_t blocks[] = {0, 1, 7, 8, 9, 67108855, 67108856, 67108857, (int64_t)1 << 24, ((int64_t)1 << 24) + 1, ((int64_t)1 << 26) + 3, 0x7fffffff};
  for (int threads : {64, 128, 256, 512, 1024})
    for (int64_t n : blocks) {
      int64_t next = 0, pieces = 0;
      bool ok = true;
      const int rc = fdm::launch_pieces(n, threads, [&](int64_t first, unsigned count) {
        ok = ok && first == next && first % 8 == 0 && count > 0 && (uint64_t)count * threads < ((uint64_t)1 << 32);
        next = first + count;
        ++pieces;
        return 0;
      });
      const int64_t fewest = (n * threads + 0xffffffffLL) >> 32;
      ok = ok && rc == 0 && next == n && pieces >= fewest && pieces <= fewest + 1 && (n * threads > 0xfffff000LL || pieces == (n > 0));
      int calls = 0;
      ok = ok && (n == 0 || (fdm::launch_pieces(n, threads, [&](int64_t, unsigned) { ++calls; return -3; }) == -3 && calls == 1));
      if (!ok) { printf("%lld blocks of %d\\n", (long long)n, threads); return 1; }
    }
  return 0;
}
""")
    binary = str(tmp_path / "pieces")
    subprocess.run([compiler, "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", binary], check=True)
    done = subprocess.run([binary], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout


@pytest.mark.parametrize("batch,sq,sk,heads", [(1 << 32, 1 << 29, 1 << 29, 1 << 30), (1 << 40, 1 << 40, 1 << 29, 1), (1 << 24, 1 << 29, 1 << 29, 1 << 30),
                                               (1 << 62, 1, 1 << 29, 4), (1 << 24, 1, 1 << 20, 32)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_window_attention_refuses_counts_past_its_numbers(batch, sq, sk, heads, head_dim):
    """Sizes whose products pass 64 bits (a count of 0 units was divided by) or 2^28 pairs: an error, and no workspace."""
    lib = N.lib()
    assert lib.fdm_attn_window_workspace_bytes(batch, sq, sk, heads, heads, head_dim, sk, 0) == 0
    assert lib.fdm_attn_window(4096, 8192, 12288, 16384, None, None, batch, sq, sk, heads, heads, head_dim, 512, 64, 512, 64, 512, 64, 512, 64, 0.125, sk, 0,
                               None, 0, None) == -2


def test_outputs_that_overlap_themselves_against_every_row():
    """All small sizes and strides of two axes, against the places themselves."""
    for B in range(4):
        for S in range(6):
            for width in (1, 2, 3):
                for bs in range(14):
                    for ts in range(14):
                        rows = [b * bs + s * ts for b in range(B) for s in range(S)]
                        places = [r + i for r in rows for i in range(width)]
                        assert N.meets_itself(width, (B, S), (bs, ts)) == (len(set(places)) < len(places)), (B, S, width, bs, ts)


def test_rotary_positions_refuses_an_output_whose_tokens_share_places(monkeypatch):
    """Strides that are each as wide as a token, but bring two tokens to one place."""
    import torch
    from fastdm_amd.kernel.operators_set import _rotary_side
    x = torch.zeros(2, 6, 128, dtype=torch.bfloat16)
    for strides in ((128, 128, 1), (256, 128, 1), (640, 128, 1), (128, 130, 1), (192, 300, 1)):
        memory = torch.zeros(4096, dtype=torch.bfloat16)
        with pytest.raises(AssertionError, match="overlaps itself"):
            _rotary_side(x, torch.as_strided(memory, (2, 6, 128), strides), 2, 6, 64, "key")
    for strides in ((768, 128, 1), (128, 256, 1), (1408, 256, 1), (800, 130, 1), (1000, 136, 1), (192, 384, 1)):      # disjoint, interleaved ones among them
        out = torch.as_strided(torch.zeros(8192, dtype=torch.bfloat16), (2, 6, 128), strides)
        assert _rotary_side(x, out, 2, 6, 64, "key")[0] is out


def test_tangents_are_refused_instead_of_lost():
    """A forward-mode dual tensor requires no gradient, but its tangent would end here without a word."""
    import torch
    import torch.autograd.forward_ad as forward_ad
    from fastdm_amd.kernel.fused import add_rms_norm
    from fastdm_amd.kernel.operators_set import rotary_positions, window_scaled_dot_product_attention
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    x, w, f = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16), RotaryFrequencies(64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: add_rms_norm(dual, None, w, 1e-6), lambda: add_rms_norm(x, dual, w, 1e-6), lambda: rotary_positions(x[None], dual[None], 64, f),
                     lambda: window_scaled_dot_product_attention(x[None], x[None], dual[None], 1, 1, 64, 4)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with pytest.raises(RuntimeError, match="tangent"), torch.no_grad():
                call()
        with pytest.raises(RuntimeError, match="GPU"):                  # no tangent: the ordinary checks
            add_rms_norm(x, None, w, 1e-6)


def test_yarn_ramp_by_hand():
    """16 elements, base 10^4, 4096 places, factor 4.  Pair x turns n times within them at x = 8 ln(4096 / (2 pi n)) / ln 10^4: n = 32 at 2.618, n = 1 at 5.628.
    The ramp runs from pair 2 (whole) to pair 6 (slowed by 4): 0, 1/4, 1/2, 3/4, 1; theta_i = 10^(-i / 2) before it."""
    from fastdm_amd.layer.embeddings import RotaryFrequencies
    kept = [1, 1, 1, 13 / 16, 10 / 16, 7 / 16, 1 / 4, 1 / 4]
    got = RotaryFrequencies(16, scaling="yarn", factor=4.0, original_length=4096)
    assert got.theta == pytest.approx([10 ** (-i / 2) * part for i, part in enumerate(kept)], rel=1e-14)
    assert got.amplitude == pytest.approx(1.138629436111989, rel=1e-15)                    # 1 + ln 4 / 10
    # 64 places: n = 32 at -0.993, so the ramp starts at pair 0; n = 1 at 2.016: it ends at pair 3
    kept = [1, 1 - 1 / 3 * 0.75, 1 - 2 / 3 * 0.75, 1 / 4, 1 / 4, 1 / 4, 1 / 4, 1 / 4]
    got = RotaryFrequencies(16, scaling="yarn", factor=4.0, original_length=64, attention_factor=1.0)
    assert got.theta == pytest.approx([10 ** (-i / 2) * part for i, part in enumerate(kept)], rel=1e-14) and got.amplitude == 1.0
