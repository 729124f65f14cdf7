"""CPU: refusals of the decoder-side operators, and the frequencies rotary_positions turns by."""
import math

import pytest
import torch

from fastdm_amd import _native as N
from fastdm_amd.layer.embeddings import RotaryFrequencies

BF16 = torch.bfloat16


def test_cpu_tensors_are_refused():
    from fastdm_amd.kernel.fused import add_rms_norm
    from fastdm_amd.kernel.operators_set import rotary_positions
    x = torch.zeros(2, 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="GPU"):
        add_rms_norm(x, x, torch.ones(64, dtype=BF16), 1e-6)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_positions(x[None], None, 64, RotaryFrequencies(64))


def c_norm(**kw):
    """fdm_add_rms_norm with made-up addresses: every call here is refused before anything is launched."""
    a = dict(out=4096, q=None, scale=None, azp=None, mode=0, x=8192, res=12288, w=16384, h=20480, rows=2, width=64, xs=64, rs=64, hs=64)
    assert set(kw) <= set(a)
    a.update(kw)
    return N.lib().fdm_add_rms_norm(a["out"], a["q"], a["scale"], a["azp"], a["mode"], a["x"], a["res"], a["w"], a["h"], a["rows"], a["width"],
                                    a["xs"], a["rs"], a["hs"], 1e-6, None)


@pytest.mark.parametrize("kw,code", [(dict(x=None), -1), (dict(w=None), -1), (dict(out=None), -1), (dict(h=None), -1), (dict(res=None), -1),
                                     (dict(rows=-1), -1), (dict(width=0), -1), (dict(mode=3), -1), (dict(mode=1), -1), (dict(mode=2, q=64, scale=64), -1),
                                     (dict(xs=63), -1), (dict(rs=63), -1), (dict(hs=63), -1), (dict(x=8193), -1), (dict(width=65537, xs=65537, rs=65537, hs=65537), -2),
                                     (dict(rows=1 << 31), -2), (dict(rows=0, x=None), 0)])
def test_add_rms_norm_c_entry_refuses(kw, code):
    assert c_norm(**kw) == code


def c_rope(**kw):
    a = dict(qo=4096, ko=8192, q=12288, k=16384, turns=20480, pos=None, pb=0, pbs=0, pts=0, B=1, S=2, hq=2, hk=1, head=64, rot=64,
             qbs=256, qts=128, kbs=128, kts=64, qobs=256, qots=128, kobs=128, kots=64, neox=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return N.lib().fdm_rope_positions(a["qo"], a["ko"], a["q"], a["k"], a["turns"], a["pos"], a["pb"], a["pbs"], a["pts"], a["B"], a["S"], a["hq"], a["hk"],
                                      a["head"], a["rot"], a["qbs"], a["qts"], a["kbs"], a["kts"], a["qobs"], a["qots"], a["kobs"], a["kots"], 1.0, a["neox"], None)


@pytest.mark.parametrize("kw,code", [(dict(turns=None), -1), (dict(turns=20484), -1), (dict(q=None), -1), (dict(ko=None), -1), (dict(q=12289), -1), (dict(rot=63), -1),
                                     (dict(rot=66), -1), (dict(rot=0), -1), (dict(head=0), -1), (dict(B=-1), -1), (dict(S=-1), -1), (dict(hq=-1), -1),
                                     (dict(pos=64, pb=2), -1), (dict(pos=68, pb=8), -1), (dict(head=512, rot=512), -2), (dict(S=1 << 31), -2),
                                     (dict(hq=1 << 20), -2), (dict(B=0, q=None), 0), (dict(S=0, turns=None), 0), (dict(hq=0, hk=0), 0)])
def test_rope_positions_c_entry_refuses(kw, code):
    assert c_rope(**kw) == code


def test_frequencies():
    f = RotaryFrequencies(8, base=10000.0)
    assert f.theta == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15) and f.amplitude == 1.0
    assert f.turns.dtype == torch.float64 and f.turns.tolist() == pytest.approx([t / (2 * math.pi) for t in f.theta], rel=1e-15)
    assert RotaryFrequencies(8, scaling="linear", factor=4.0).theta == pytest.approx([t / 4 for t in f.theta])
    ntk = RotaryFrequencies(8, scaling="ntk", factor=4.0).theta
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(f.theta[-1] / 4)
    own = RotaryFrequencies(4, frequencies=[0.5, 0.25], attention_factor=2.0)
    assert own.theta == [0.5, 0.25] and own.amplitude == 2.0


def test_yarn_keeps_the_fast_pairs_and_slows_the_others():
    d, L, s = 128, 4096, 16.0
    plain, got = RotaryFrequencies(d), RotaryFrequencies(d, scaling="yarn", factor=s, original_length=L)
    assert got.amplitude == pytest.approx(0.1 * math.log(s) + 1)
    for a, b in zip(plain.theta, got.theta):
        turns = L * a / (2 * math.pi)
        if turns > 40:
            assert b == pytest.approx(a)
        elif turns < 0.8:
            assert b == pytest.approx(a / s)
        assert a / s * (1 - 1e-12) <= b <= a * (1 + 1e-12)


def test_wavelength_blends_between_its_two_ends():
    L, s = 8192, 8.0
    plain, got = RotaryFrequencies(128, base=500000.0), RotaryFrequencies(128, base=500000.0, scaling="wavelength", factor=s, original_length=L)
    for a, b in zip(plain.theta, got.theta):
        length = 2 * math.pi / a
        if length <= L / 4:
            assert b == pytest.approx(a)
        elif length >= L:
            assert b == pytest.approx(a / s)
        else:
            m = (L / length - 1) / 3
            assert b == pytest.approx((1 - m) * a / s + m * a)


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=258), dict(rotary_dim=64, scaling="other"), dict(rotary_dim=64, scaling="yarn", factor=2.0),
                                dict(rotary_dim=64, scaling="wavelength", factor=2.0), dict(rotary_dim=2, scaling="ntk", factor=2.0), dict(rotary_dim=64, base=1.0),
                                dict(rotary_dim=64, factor=0.0, scaling="linear"), dict(rotary_dim=4, frequencies=[1.0]),
                                dict(rotary_dim=4, frequencies=[1.0, 0.5], scaling="linear", factor=2.0),
                                dict(rotary_dim=64, scaling="yarn", factor=2.0, original_length=4096, beta_fast=1.0, beta_slow=2.0),
                                dict(rotary_dim=64, scaling="wavelength", factor=2.0, original_length=4096, low_factor=4.0)])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        RotaryFrequencies(**kw)


def c_window(**kw):
    a = dict(o=4096, q=8192, k=12288, v=16384, ql=None, kl=None, B=1, sq=4, sk=8, hq=2, hk=1, D=64, qbs=512, qts=128, kbs=512, kts=64, vbs=512, vts=64, obs=512, ots=128,
             scale=0.125, window=4, sinks=0, ws=None, wsb=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return N.lib().fdm_attn_window(a["o"], a["q"], a["k"], a["v"], a["ql"], a["kl"], a["B"], a["sq"], a["sk"], a["hq"], a["hk"], a["D"], a["qbs"], a["qts"], a["kbs"], a["kts"],
                                   a["vbs"], a["vts"], a["obs"], a["ots"], a["scale"], a["window"], a["sinks"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,code", [(dict(o=None), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(q=8200), -1), (dict(kts=63), -1), (dict(vbs=-512), -1),
                                     (dict(ql=2), -1), (dict(kl=6), -1), (dict(hq=3, hk=2), -1), (dict(hk=0), -1), (dict(window=0), -1), (dict(sinks=-1), -1),
                                     (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(B=-1), -1),
                                     (dict(D=96), -2), (dict(sk=(1 << 29) + 1), -2), (dict(sq=(1 << 29) + 1), -2), (dict(sq=0, q=None), 0), (dict(B=0, o=None), 0),
                                     (dict(sq=1, sk=100000, window=100000), -1), (dict(sq=1, sk=100000, window=100000, ws=64, wsb=64), -1)])
def test_window_attention_c_entry_refuses(kw, code):
    assert c_window(**kw) == code


def test_window_attention_workspace_is_for_few_long_rows_alone():
    need = N.lib().fdm_attn_window_workspace_bytes
    assert need(1, 1, 100000, 8, 8, 128, 100000, 0) > 0
    assert need(64, 1, 100, 8, 8, 128, 100, 0) == 0 and need(1, 65536, 65536, 32, 8, 128, 4096, 4) == 0
    assert need(0, 1, 1, 1, 1, 64, 1, 0) == 0 and need(1, 1, 1, 3, 2, 64, 1, 0) == 0


def test_window_attention_refuses_cpu_tensors():
    from fastdm_amd.kernel.operators_set import window_scaled_dot_product_attention
    x = torch.zeros(1, 4, 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="GPU"):
        window_scaled_dot_product_attention(x, x, x, 1, 1, 64, 2)


@pytest.mark.parametrize("kw,code", [(dict(head=1032, rot=64), -2), (dict(hq=65536, hk=1, head=64), -2)])
def test_rope_positions_c_entry_refuses_what_its_numbers_do_not_hold(kw, code):
    assert c_rope(**kw) == code


def test_launch_goes_to_the_tensors_device(monkeypatch):
    """A kernel is launched with its tensors' GPU as the current device and on that GPU's stream, whichever was current."""
    seen, current = [], [0]

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(N, "_current_device", lambda: current[0])
    monkeypatch.setattr(N, "stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", device)

    def entry(*args):
        seen.append((current[0], args))
        return 0

    N.launch("x", 0, entry, 1)
    N.launch("x", 3, entry, 2)
    assert seen == [(0, (1, 100)), (3, (2, 103))] and current[0] == 0
    with pytest.raises(RuntimeError, match="x failed: unsupported"):
        N.launch("x", 0, lambda *a: -2)


def test_outputs_across_inputs_are_told_from_slices_and_from_in_place():
    m = torch.zeros(8, 96, dtype=BF16)
    a = m[:4, :32]
    assert not N.crosses(a, m[:4, :32]) and N.crosses(a, m[:4, :32], same=True) and not N.crosses(a, a) and N.crosses(a, a, same=True)      # in place
    assert not N.crosses(a, m[:4, 32:64]) and not N.crosses(a, m[1:5, 32:64]) and not N.crosses(a, m[4:, :32])                              # beside, behind
    assert N.crosses(a, m[1:5, :32]) and N.crosses(m[1:5, :32], a) and N.crosses(a, m[:4, 16:48]) and N.crosses(m[:4, 16:48], a)            # shifted
    assert N.crosses(a, m.view(-1)[:256].view(4, 64)[:, :32]) and not N.crosses(a, torch.zeros(4, 32, dtype=BF16))                         # other strides
    assert N.crosses(m[:1, :32], m[:1, 16:48]) and not N.crosses(m[:1, :32], m[:1, 32:64]) and not N.crosses(m[:0], m[:0], same=True)              # one row, none
    b = torch.zeros(2, 6, 96, dtype=BF16)
    assert not N.crosses(b[..., :64], b[..., 64:], same=True) and N.crosses(b[..., :64], b[..., 32:]) and N.crosses(b[:, :5, :64], b[:, 1:, :64])
    assert not N.crosses(b[:, :3, :64], b[:, 3:, 64:]) and not N.crosses(b[:1, :, :64], b[1:, :, :64])
    assert not N.crosses(b[:, :3, :64], b[:, 3:, :64], same=True) and N.crosses(b[:, :4, :64], b[:, 2:, :64])       # tokens in front of others'


def test_outputs_across_inputs_against_every_row():
    """All pairs of slices of a small tensor, against the addresses themselves."""
    import itertools
    base = torch.zeros(3, 4, 6, dtype=BF16)
    places = torch.arange(base.numel()).view(3, 4, 6)
    cuts = [(slice(i, i + B), slice(j, j + S), slice(c, c + W)) for B, S, W in ((2, 2, 3), (1, 3, 2), (2, 1, 4), (1, 1, 6))
            for i in range(4 - B) for j in range(5 - S) for c in range(7 - W)]
    for x, y in itertools.product(cuts, cuts):
        a, out = base[x], base[y]
        if a.shape[:2] == out.shape[:2]:
            share = bool(set(places[x].flatten().tolist()) & set(places[y].flatten().tolist()))
            assert N.crosses(a, out, same=True) == share, (x, y)
            assert N.crosses(a, out) == (share and x != y), (x, y)
    other = base.view(4, 3, 6)
    assert N.crosses(base[:2, :2], other[:2, :2]) and not N.crosses(base[:1, :2], other[3:, :2])
