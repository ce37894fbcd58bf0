"""CPU tests of the steps between projections: refusals, argument checks of the C entry points, rotary frequencies."""
import ctypes
import math

import pytest
import torch

from sacq_b200 import _lib, attention_packed, residual_norm_quantize_rows, rotary_frequencies, rotate_heads


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_steps_refuse_cpu_tensors_and_other_types():
    cu, pos, freq = torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.ones(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        attention_packed(_bf(4, 2, 64), _bf(4, 2, 64), _bf(4, 2, 64), cu)
    with pytest.raises(ValueError, match="CUDA"):
        rotate_heads(_bf(4, 2, 64), _bf(4, 2, 64), pos, freq)
    with pytest.raises(TypeError, match="CUDA"):
        residual_norm_quantize_rows(_bf(4, 64), _bf(4, 64))
    for bad in (torch.zeros(4, 2, 64), torch.zeros(4, 2, 64, dtype=torch.float16), _bf(4, 128), None, [1]):
        with pytest.raises(TypeError):
            attention_packed(bad, _bf(4, 2, 64), _bf(4, 2, 64), cu)
        with pytest.raises(TypeError):
            rotate_heads(bad, None, pos, freq)
        with pytest.raises(TypeError):
            residual_norm_quantize_rows(bad, _bf(4, 64))
    with pytest.raises(ValueError, match="layout"):
        rotate_heads(_bf(4, 2, 64), None, pos, freq, layout="quarter")
    with pytest.raises(ValueError, match="norm"):
        residual_norm_quantize_rows(_bf(4, 64), _bf(4, 64), norm="batch")
    with pytest.raises(ValueError, match="norm"):
        residual_norm_quantize_rows(_bf(4, 64), _bf(4, 64), post_norm="batch")


def _filled(cls, **values):
    d = cls(struct_size=ctypes.sizeof(cls))
    for n, v in values.items():
        setattr(d, n, v)
    return d


def test_c_entry_points_check_their_arguments():
    lib = _lib.load()
    one = ctypes.c_void_p(256)

    def attention(**kw):
        base = dict(q=one, k=one, v=one, out=one, cu_q=one, cu_k=one, tokens_q=4, tokens_k=4, sequences=1, heads=4, kv_heads=2, head_dim=64, scale=1.0,
                    q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, out_token=256, out_head=64)
        return lib.sacq_attention_packed(ctypes.byref(_filled(_lib.AttentionDesc, **{**base, **kw})), None)

    assert lib.sacq_attention_packed(None, None) == -1 and lib.sacq_attention_workspace_bytes(None) < 0
    assert attention(struct_size=8) == -1 and "struct_size" in _lib.last_error()
    for kw in (dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(head_dim=0), dict(tokens_q=-1), dict(tokens_k=-1), dict(sequences=-1), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_q=None),
               dict(cu_k=None)):
        assert attention(**kw) == -1, kw
    for kw in (dict(head_dim=257), dict(tokens_q=2 ** 31), dict(tokens_k=2 ** 31)):
        assert attention(**kw) == -2, kw
    assert attention(tokens_q=0) == 0 and attention(sequences=0) == 0

    def rotary(**kw):
        heads = dict(in_=one, out=one, in_token=128, in_head=64, out_token=128, out_head=64, heads=2)
        d = _filled(_lib.RotaryDesc, layout=0, tokens=4, head_dim=64, rotary_dim=64, positions=one, position_bytes=4, amplitude=1.0, inv_freq=one)
        for name in ("q", "k"):
            for n, v in {**heads, **kw.pop(name, {})}.items():
                setattr(getattr(d, name), n, v)
        for n, v in kw.items():
            setattr(d, n, v)
        return lib.sacq_rotate_heads(ctypes.byref(d), None)

    assert lib.sacq_rotate_heads(None, None) == -1
    for kw in (dict(struct_size=4), dict(tokens=-1), dict(head_dim=0), dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=66), dict(layout=2),
               dict(position_bytes=2), dict(positions=None), dict(inv_freq=None), dict(q=dict(in_=None)), dict(k=dict(out=None)), dict(q=dict(heads=-1))):
        assert rotary(**kw) == -1, kw
    assert rotary(head_dim=8192, rotary_dim=64) == -2
    assert rotary(tokens=0) == 0 and rotary(q=dict(heads=0), k=dict(heads=0)) == 0

    def norm(**kw):
        base = dict(norm=1, post_norm=0, eps=1e-6, residual_scale=1.0, M=2, K=64, branch=one, residual=one, branch_pitch=64, residual_pitch=64,
                    residual_out=one, q_out=one, scale_out=one)
        return lib.sacq_residual_norm(ctypes.byref(_filled(_lib.ResidualNormDesc, **{**base, **kw})), None)

    assert lib.sacq_residual_norm(None, None) == -1
    for kw in (dict(struct_size=1), dict(M=-1), dict(K=0), dict(branch=None), dict(residual=None), dict(residual_out=None), dict(scale_out=None),
               dict(q_out=None, scale_out=None), dict(norm=0), dict(norm=3), dict(post_norm=3), dict(post_weight=one), dict(mod_scale=one),
               dict(vector_rows=one, gate=one), dict(branch_pitch=63), dict(residual_pitch=63), dict(eps=-1.0), dict(eps=math.nan)):
        assert norm(**kw) == -1, kw
    assert norm(M=0) == 0
    assert norm(K=40000, branch_pitch=40000, residual_pitch=40000) == -2


def test_rotary_frequencies():
    freq, amp = rotary_frequencies(8, device="cpu")
    assert amp == 1.0 and freq.dtype == torch.float64
    assert torch.allclose(freq, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(rotary_frequencies(8, scaling={"kind": "linear", "factor": 4.0}, device="cpu")[0], freq / 4)
    base, _ = rotary_frequencies(8, scaling={"kind": "base", "factor": 4.0}, device="cpu")
    assert float(base[0]) == 1.0 and math.isclose(float(base[-1]), float(freq[-1]) / 4, rel_tol=1e-12)
    freq, _ = rotary_frequencies(128, device="cpu")
    turns = 4096 * freq / (2 * math.pi)
    yarn, amp = rotary_frequencies(128, scaling={"kind": "yarn", "factor": 16.0, "original": 4096}, device="cpu")
    assert math.isclose(amp, 0.1 * math.log(16) + 1)
    # one index of slack at either end of the ramp
    assert torch.equal(yarn[:-1][turns[1:] >= 32], freq[:-1][turns[1:] >= 32])
    assert torch.allclose(yarn[1:][turns[:-1] < 1], freq[1:][turns[:-1] < 1] / 16, rtol=1e-12)
    assert bool((yarn <= freq).all()) and bool((yarn >= freq / 16 * (1 - 1e-12)).all()) and bool((yarn.diff() < 0).all())
    assert rotary_frequencies(128, scaling={"kind": "yarn", "factor": 2.0, "original": 64, "amplitude": 1.5}, device="cpu")[1] == 1.5
    band, amp = rotary_frequencies(128, scaling={"kind": "wavelength", "factor": 8.0, "original": 4096}, device="cpu")
    assert amp == 1.0 and torch.equal(band[turns >= 4], freq[turns >= 4]) and torch.allclose(band[turns <= 1], freq[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    keep = (turns[mid] - 1) / 3
    assert torch.allclose(band[mid], freq[mid] * keep + freq[mid] / 8 * (1 - keep), rtol=1e-12)
    for dim, kw in ((7, {}), (0, {}), (8, {"base": 1.0}), (8, {"scaling": {"kind": "other", "factor": 2.0}}), (8, {"scaling": {"kind": "linear"}}),
                    (8, {"scaling": {"kind": "linear", "factor": 0.5}}), (8, {"scaling": {"kind": "yarn", "factor": 2.0}}),
                    (8, {"scaling": {"kind": "linear", "factor": 2.0, "original": 3}}), (2, {"scaling": {"kind": "base", "factor": 2.0}}),
                    (8, {"scaling": {"kind": "yarn", "factor": 2.0, "original": 4096, "beta_fast": 1.0, "beta_slow": 2.0}}),
                    (8, {"scaling": {"kind": "wavelength", "factor": 2.0, "original": 4096, "low": 4.0, "high": 4.0}})):
        with pytest.raises(ValueError):
            rotary_frequencies(dim, device="cpu", **kw)


def test_views_overlap_where_they_share_elements():
    overlaps = _lib.native().overlaps
    x = torch.zeros(6, 12, 8)
    apart = ((x[:, :4], x[:, 4:8]), (x[:3], x[3:]), (x[:, ::2], x[:, 1::2]), (x[:, :, :4], x[:, :, 4:]), (x[::2], x[1::2]), (x[:, 3:5], x[:, 5:]),
             (x[:, 8:, :2], x[:, :8, 1:]), (x[:0], x), (x[:, :1], x[:, 1:]), (x[:1, ::2], x[:1, 1::2]))
    shared = ((x, x), (x[:, :5], x[:, 4:8]), (x[:4], x[3:]), (x[:, ::2], x[:, ::3]), (x[:, :, :5], x[:, :, 4:]), (x[1], x[:, 3:4]), (x[:, 1:2], x[:, :4]))
    for pairs, want in ((apart, False), (shared, True)):
        for a, b in pairs:
            assert overlaps(a, (b,)) is want and overlaps(b, (a,)) is want and overlaps(a, (None, b)) is want
    # against the elements themselves, over small views; what shares must be found, what does not may be called shared
    storage, found = torch.arange(400), 0
    rng = torch.Generator().manual_seed(5)
    for _ in range(2000):
        n = lambda hi: int(torch.randint(1, hi, (1,), generator=rng))
        views = [storage.as_strided((n(4), n(4), n(4)), (n(30), n(12), 1), n(60)) for _ in range(2)]
        share = bool(set(views[0].flatten().tolist()) & set(views[1].flatten().tolist()))
        found += share
        assert overlaps(views[0], (views[1],)) or not share
    assert 100 < found < 1900
