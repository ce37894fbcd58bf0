"""Attention over packed sequences, rotary positions and the norms around a block against plain float64 evaluations.

Tolerances are sums of the roundings a kernel makes: half a step of a bf16 result or weight is 2^-8 of the value, of an fp32
operation 2^-24, of e4m3 2^-4; a sum of n fp32 terms is off by at most n 2^-24 of the sum of their magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = 2.0 ** -8, 2.0 ** -24
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _needs_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, at=0.0, by=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * by + at).to(torch.bfloat16)


def _offsets(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


# ----------------------------------------------------------------------------- attention

def _attention_reference(q, k, v, lq, lk, causal, scale=None):
    """(out, lse, bound of out, bound of lse) in float64, sequence by sequence.  Only keys that a query sees are looked at."""
    d, g = q.shape[2], q.shape[1] // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -INF, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    aq = ak = 0
    for nq, nk in zip(lq, lk):
        if nq and nk:
            qs = q[aq:aq + nq].double().transpose(0, 1)
            ks, vs = (t[ak:ak + nk].double().transpose(0, 1).repeat_interleave(g, 0) for t in (k, v))
            s = qs @ ks.transpose(1, 2) * scale
            # a score is a sum of d products in fp32, scaled and shifted by the maximum; exp and its argument: 2^-20
            off = (qs.abs() @ ks.abs().transpose(1, 2) * scale) * (d + 8) * F32
            seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
            if causal:
                seen = seen.tril(nk - nq)
            s = s.masked_fill(~seen, -INF)
            off = (off + s.abs() * 4 * F32).masked_fill(~seen, 0.0)
            le = torch.logsumexp(s, 2)
            p = (s - le.masked_fill(le == -INF, 0.0)[..., None]).exp()
            spread = (p @ vs.abs()).transpose(0, 1)                     # sum p |v|
            worst = off.amax(2).transpose(0, 1)[..., None]
            o = p @ vs
            o = o.transpose(0, 1)
            out[aq:aq + nq], lse[aq:aq + nq] = o, le.transpose(0, 1)
            # weights rounded to bf16, fp32 sums of nk terms, errors of the scores on weights and their sum, the result rounded to bf16
            rel = BF + nk * F32 + 2 * worst + 2.0 ** -20
            tol[aq:aq + nq] = spread.nan_to_num(0.0) * rel * 1.01 + o.abs().nan_to_num(0.0) * BF * 1.01 + 1e-30
            tol_lse[aq:aq + nq] = worst[..., 0] + (nk + 8) * F32 + 2.0 ** -20 + le.transpose(0, 1).abs().nan_to_num(0.0, posinf=0.0) * 4 * F32
        aq, ak = aq + nq, ak + nk
    return out, lse, tol, tol_lse


def _check_attention(got, lse, ref):
    out, le, tol, tol_le = ref
    got, lse = got.double(), lse.double()
    assert bool(torch.isfinite(got).all())
    bad = (got - out).abs() - tol
    assert float(bad.max()) <= 0, (float(bad.max()), (bad > 0).nonzero()[:4].tolist())
    none = le == -INF
    assert torch.equal(lse == -INF, none) and bool((got[none] == 0).all())
    off = (lse - le).abs()[~none] - tol_le[~none]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def _attend(lq, lk, heads, kv_heads, dim, causal, seed=0, by=1.5, scale=None):
    from sacq_b200 import attention_packed
    gen = _gen(seed)
    q = _randn(gen, sum(lq), heads, dim, by=by)
    k, v = (_randn(gen, sum(lk), kv_heads, dim, by=by) for _ in range(2))
    got, lse = attention_packed(q, k, v, _offsets(lq), _offsets(lk), causal=causal, scale=scale, return_lse=True)
    assert got.dtype == torch.bfloat16 and got.shape == q.shape and lse.dtype == torch.float32
    _check_attention(got, lse, _attention_reference(q, k, v, lq, lk, causal, scale))


@pytest.mark.parametrize("causal", (False, True))
@pytest.mark.parametrize("lengths", ([1], [2, 1, 3], [16], [63, 64, 65], [127, 1, 128, 129], [255, 256, 257], [300, 0, 41], [513, 700]))
def test_attention_of_a_prompt(lengths, causal):
    _attend(lengths, lengths, 4, 2, 128, causal)


@pytest.mark.parametrize("heads,kv_heads,dim", ((12, 12, 128), (16, 16, 64), (8, 1, 128), (6, 2, 96), (9, 3, 64), (4, 4, 80), (7, 1, 8), (12, 1, 16),
                                                (128, 1, 64), (5, 5, 72), (2, 1, 112), (3, 1, 36), (2, 2, 200), (1, 1, 1), (4, 2, 256)))
@pytest.mark.parametrize("causal", (False, True))
def test_attention_head_layouts(heads, kv_heads, dim, causal):
    _attend([70, 150, 5], [70, 150, 5], heads, kv_heads, dim, causal)


@pytest.mark.parametrize("lq,lk", (([16, 16], [300, 270]), ([1, 1, 1], [1, 500, 4097]), ([1], [20000]), ([3, 7], [130, 128]), ([200, 5], [7, 130]),
                                   ([130, 4, 9], [0, 0, 40]), ([40, 0, 3], [30, 50, 0]), ([150], [1]), ([2, 1, 300], [6000, 31, 2500])))
@pytest.mark.parametrize("causal", (False, True))
def test_attention_to_keys_of_other_lengths(lq, lk, causal):
    # causal with fewer keys than queries: the first queries see none
    _attend(lq, lk, 4, 2, 128, causal)
    _attend(lq, lk, 3, 3, 64, causal, seed=1)


@pytest.mark.parametrize("lq,lk,heads,kv_heads", (([100, 100], [4000, 3001], 4, 4), ([130], [6000], 2, 2), ([300, 3], [5100, 129], 3, 1), ([70, 1, 65], [5000, 0, 140], 4, 2),
                                                  ([2300], [2300], 1, 1), ([5, 1], [7000, 200], 4, 2)))
@pytest.mark.parametrize("dim", (128, 64, 80, 40))
@pytest.mark.parametrize("causal", (False, True))
def test_attention_of_few_queries_to_many_keys(lq, lk, heads, kv_heads, dim, causal):
    """Keys in chunks of several tiles, one and two tiles of queries; rows that a chunk holds nothing for."""
    _attend(lq, lk, heads, kv_heads, dim, causal, seed=7)


@pytest.mark.parametrize("dim", (128, 64))
def test_attention_of_chunks_keeps_what_is_not_seen_out(dim):
    from sacq_b200 import attention_packed
    gen = _gen(9)
    q, (k, v) = _randn(gen, 90, 2, dim), (_randn(gen, 5000, 2, dim) for _ in range(2))
    cu_q, cu_k = _offsets([90]), _offsets([4700])
    want = attention_packed(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    for t in (k, v):
        t[4700:] = NAN
        t[4690:4700] = INF                   # seen by the last queries only
    got = attention_packed(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    # rows that see none of them are made again key by key there: other roundings of the same sums
    assert float((got[0][:80].double() - want[0][:80].double()).abs().max()) <= 2 * BF * float(want[0].abs().max())
    assert float((got[1][:80] - want[1][:80]).abs().max()) <= 2 * 4700 * F32          # two fp32 sums of as many weights
    assert not bool(torch.isfinite(got[0][80:].float()).all(dim=-1).any())


def test_attention_of_many_sequences():
    lengths = [(7 * i) % 40 for i in range(300)]
    _attend(lengths, lengths, 2, 1, 64, True)
    _attend([1] * 300, [(37 * i) % 700 for i in range(300)], 4, 2, 128, True)


@pytest.mark.parametrize("by", (0.01, 6.0, 40.0))
def test_attention_of_flat_and_peaked_scores(by):
    _attend([200, 77], [200, 77], 4, 2, 128, True, by=by)
    _attend([200, 77], [1200, 77], 2, 2, 64, False, by=by)


def test_attention_rising_scores():
    """Each tile of keys outdoes the ones in front of it, so that every step rescales what it has."""
    from sacq_b200 import attention_packed
    gen = _gen(3)
    n = 700
    q, k, v = (_randn(gen, n, 2, 128) for _ in range(3))
    k = (k.float() * 0.1 + q[:1].float() * torch.linspace(0, 4, n, device="cuda")[:, None, None]).to(torch.bfloat16)
    q = (q[:1].float() + q.float() * 0.05).to(torch.bfloat16)
    for causal in (False, True):
        got, lse = attention_packed(q, k, v, _offsets([n]), causal=causal, return_lse=True)
        _check_attention(got, lse, _attention_reference(q, k, v, [n], [n], causal))


@pytest.mark.parametrize("scale", (1.0, 0.3, 1e-4))
def test_attention_scale(scale):
    _attend([90, 33], [90, 33], 2, 2, 64, True, by=1.0, scale=scale)


@pytest.mark.parametrize("dim", (64, 128))
def test_attention_reads_views_where_they_lie(dim):
    from sacq_b200 import attention_packed
    gen = _gen(4)
    lengths = [140, 33, 250]
    t, h, hk = sum(lengths), 6, 2
    fused = _randn(gen, t, (h + 2 * hk) * dim + 8)
    q, k, v = (fused[:, a * dim:(a + n) * dim].view(t, n, dim) for a, n in ((0, h), (h, hk), (h + hk, hk)))
    out = torch.full((t + 5, h, 2 * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = attention_packed(q, k, v, _offsets(lengths), causal=True, out=out[2:t + 2, :, dim:], return_lse=True)
    assert got.data_ptr() == out[2:t + 2, :, dim:].data_ptr()
    _check_attention(got, lse, _attention_reference(q, k, v, lengths, lengths, True))
    assert bool((out[:2] == 7).all()) and bool((out[t + 2:] == 7).all()) and bool((out[..., :dim] == 7).all())
    # heads first, an inner stride that is not one, a head stride that is not a multiple of 8 elements
    for make in (lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda x: torch.nn.functional.pad(x, (0, 3))[..., :dim], lambda x: torch.nn.functional.pad(x.reshape(t, -1), (1, 0))[:, 1:].view(x.shape)):
        again = attention_packed(make(q), make(k), make(v), _offsets(lengths), causal=True)
        ref = _attention_reference(q, k, v, lengths, lengths, True)
        assert float(((again.double() - ref[0]).abs() - ref[2]).max()) <= 0
    # one key-value row for every token
    one = k[:1].expand(t, hk, dim)
    again, lse = attention_packed(q, one, one, _offsets(lengths), causal=True, return_lse=True)
    _check_attention(again, lse, _attention_reference(q, one, one, lengths, lengths, True))


@pytest.mark.parametrize("heads,dim", (((4, 2), 128), ((2, 2), 64), ((2, 1), 36)))
@pytest.mark.parametrize("value", (NAN, INF, -INF, 3e38))
def test_attention_keeps_what_is_not_seen_out(value, heads, dim):
    """Rows of no sequence, of other sequences and of later tokens may hold anything."""
    from sacq_b200 import attention_packed
    gen = _gen(5)
    lengths = [130, 3, 60]
    front, behind = 9, 100
    t = front + sum(lengths) + behind
    q, k, v = (_randn(gen, t, n, dim) for n in (heads[0], heads[1], heads[1]))
    cu = (_offsets(lengths) + front).to(torch.int32)
    real = slice(front, t - behind)
    ref = _attention_reference(q[real], k[real], v[real], lengths, lengths, True)
    for x in (q, k, v):
        x[:front], x[t - behind:] = value, value
    out = torch.full_like(q, 3.0)
    lse = attention_packed(q, k, v, cu, causal=True, out=out, return_lse=True)[1]
    _check_attention(out[real], lse[real], ref)
    assert bool((out[:front] == 3).all()) and bool((out[t - behind:] == 3).all())
    # the middle sequence and the last tokens of the first
    k2, v2 = k.clone(), v.clone()
    hidden = slice(front + 120, front + 133)
    k2[hidden], v2[hidden] = value, value
    attention_packed(q, k2, v2, cu, causal=True, out=out)
    clean = list(range(0, 120)) + list(range(133, sum(lengths)))
    bad = (out[real][clean].double() - ref[0][clean]).abs() - ref[2][clean]
    assert float(bad.max()) <= 0


def test_attention_of_infinities_that_are_seen():
    """A visible NaN or infinity reaches the rows that see it as it does in the formula."""
    from sacq_b200 import attention_packed
    gen = _gen(6)
    q, k, v = (_randn(gen, 40, 1, 64) for _ in range(3))
    v[30, 0, 5], v[35, 0, 6] = INF, NAN
    out = attention_packed(q, k, v, _offsets([40]), causal=True)
    assert bool(torch.isfinite(out[:30]).all())
    assert bool((out[30:, 0, 5] == INF).all()) and bool(torch.isfinite(out[30:35, 0, 6]).all()) and bool(out[35:, 0, 6].isnan().all())
    k[20] = NAN
    out = attention_packed(q, k, v, _offsets([40]), causal=True)
    assert bool(torch.isfinite(out[:20]).all()) and bool(out[20:].isnan().all())


def test_attention_is_the_same_twice_and_does_not_depend_on_the_batch():
    from sacq_b200 import attention_packed
    gen = _gen(7)
    lengths = [300, 120, 4, 700]
    q, k, v = (_randn(gen, sum(lengths), n, 128) for n in (8, 4, 4))
    a, b = (attention_packed(q, k, v, _offsets(lengths), causal=True) for _ in range(2))
    assert torch.equal(a, b)
    at = 0
    for n in lengths:
        one = attention_packed(q[at:at + n], k[at:at + n], v[at:at + n], _offsets([n]), causal=True)
        ref = _attention_reference(q[at:at + n], k[at:at + n], v[at:at + n], [n], [n], True)
        assert float(((one.double() - ref[0]).abs() - ref[2]).max()) <= 0
        assert float((one.double() - a[at:at + n].double()).abs().sub(2 * ref[2]).max()) <= 0
        at += n


def test_attention_offsets_that_leave_the_tensors():
    """Offsets are cut to the tensors, and a sequence that ends in front of its beginning is empty."""
    from sacq_b200 import attention_packed
    gen = _gen(8)
    q, k, v = (_randn(gen, 100, 2, 64) for _ in range(3))
    cu = torch.tensor([-5, 40, 1000], dtype=torch.int32, device="cuda")
    out, lse = attention_packed(q, k, v, cu, return_lse=True)
    _check_attention(out, lse, _attention_reference(q, k, v, [40, 60], [40, 60], False))
    out = torch.full_like(q, 2.0)
    attention_packed(q, k, v, torch.tensor([60, 20, 100], dtype=torch.int32, device="cuda"), out=out)
    ref = _attention_reference(q[20:], k[20:], v[20:], [80], [80], False)
    assert float(((out[20:].double() - ref[0]).abs() - ref[2]).max()) <= 0
    assert bool((out[:20] == 2).all())


def test_attention_empty_calls():
    from sacq_b200 import attention_packed
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    assert attention_packed(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), _offsets([])).shape == (0, 4, 64)
    out, lse = attention_packed(z(5, 4, 64) + 1, z(0, 2, 64), z(0, 2, 64), _offsets([5]), _offsets([0]), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -INF).all())
    out = torch.full((5, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    attention_packed(z(5, 4, 64), z(3, 2, 64), z(3, 2, 64), _offsets([]), out=out)
    assert bool((out == 9).all())


# ----------------------------------------------------------------------------- rotary positions

def _rotary_reference(x, positions, inv_freq, layout, amplitude):
    r = 2 * inv_freq.numel()
    x = x.double()
    angle = positions.double()[:, None, None] * inv_freq
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    i = torch.arange(r // 2, device=x.device)
    first, second = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y, tol = x.clone(), torch.zeros_like(x)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    # the angle rounded to 2^-26 turns (2^-23.3 radians), sine and cosine to 2 ulp, three fp32 operations; the result to bf16.  In double the
    # kernel rounds inv_freq / 2 pi and its product with the position, this reference its own product: 3 x 2^-53 of the angle, which at
    # 2^33 positions is 2.9e-6 radians and more than all the rest
    small = (a.abs() + b.abs()) * abs(amplitude) * (2.0 ** -20 + angle.abs() * 3 * 2.0 ** -53)
    tol[..., first] = tol[..., second] = small
    return y, torch.where(tol > 0, tol * 1.01 + y.abs() * BF, 0.0)


@pytest.mark.parametrize("layout", ("half", "interleaved"))
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", ((1, 16, 8, 128, 128), (3, 12, 12, 128, 64), (257, 6, 2, 96, 96), (1000, 4, 4, 80, 40), (37, 1, 1, 64, 2),
                                                              (5, 2, 1, 36, 20), (64, 3, 3, 7, 6), (19, 128, 1, 64, 64), (2, 2, 2, 512, 256), (700, 32, 8, 128, 32), (800, 1, 1, 4096, 4096)))
def test_rotary(layout, tokens, heads, kv_heads, dim, rotary):
    from sacq_b200 import rotary_frequencies, rotate_heads
    gen = _gen(tokens)
    q, k = _randn(gen, tokens, heads, dim), _randn(gen, tokens, kv_heads, dim)
    freq, _ = rotary_frequencies(rotary)
    for dtype, most, amplitude in ((torch.int32, 4096, 1.0), (torch.int64, 2 ** 33, 1.25)):
        pos = torch.randint(0, most, (tokens,), generator=gen, device="cuda", dtype=dtype)
        pos[0] = -3
        for got, x in zip(rotate_heads(q, k, pos, freq, layout=layout, amplitude=amplitude), (q, k)):
            ref, tol = _rotary_reference(x, pos, freq, layout, amplitude)
            assert got.dtype == torch.bfloat16 and float(((got.double() - ref).abs() - tol).max()) <= 0


@pytest.mark.parametrize("layout", ("half", "interleaved"))
def test_rotary_views_and_in_place(layout):
    from sacq_b200 import rotary_frequencies, rotate_heads
    gen = _gen(1)
    t, d = 300, 128
    fused = _randn(gen, t, 6 * d)
    freq, amp = rotary_frequencies(96, scaling={"kind": "yarn", "factor": 8.0, "original": 4096})
    pos = torch.arange(t, device="cuda", dtype=torch.int32) + 70000
    heads = [fused[:, :4 * d].view(t, 4, d), fused[:, 4 * d:5 * d].view(t, 1, d)]
    refs = [_rotary_reference(x, pos, freq, layout, amp) for x in heads]
    fresh = rotate_heads(*heads, pos, freq, layout=layout, amplitude=amp)
    v = fused[:, 5 * d:].clone()
    assert rotate_heads(*heads, pos, freq, layout=layout, amplitude=amp, out=tuple(heads))[0].data_ptr() == fused.data_ptr()
    for x, f, (ref, tol) in zip(heads, fresh, refs):
        assert torch.equal(x, f) and float(((x.double() - ref).abs() - tol).max()) <= 0
    assert torch.equal(v, fused[:, 5 * d:])
    # odd strides take the kernel for single elements; an inner stride and no key heads
    odd = torch.nn.functional.pad(fresh[0], (0, 1))[..., :d]
    again = rotate_heads(odd, None, pos, freq, layout=layout)
    ref, tol = _rotary_reference(fresh[0], pos, freq, layout, 1.0)
    assert again[1] is None and float(((again[0].double() - ref).abs() - tol).max()) <= 0
    flipped = fresh[0].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rotate_heads(flipped, None, pos, freq, layout=layout)[0],
                       rotate_heads(fresh[0], None, pos, freq, layout=layout)[0])
    empty = rotate_heads(fresh[0][:0], fresh[1][:0], pos[:0], freq)
    assert empty[0].shape == (0, 4, d) and empty[1].shape == (0, 1, d)


# ----------------------------------------------------------------------------- norms around a block

def _norm_reference(branch, residual, p, norm, post, eps, scale):
    """(r, h, bound of r, bound of h) in float64; p: the vectors, as rows."""
    one = lambda n, x: x if p[n] is None else p[n].double()  # noqa: E731
    k = branch.shape[1]

    def normed(x, kind, w, b, off):
        """norm(x) w + b, and its error for an error `off` of x."""
        c = x - x.mean(1, keepdim=True) if kind == "layer" else x
        rstd = (c.square().mean(1, keepdim=True) + eps).rsqrt()
        y = c * rstd * w
        # the mean: k terms, and its share of off; the mean square: k terms, half of it on rstd, and the share of off on it
        shift = k * F32 * x.abs().mean(1, keepdim=True) + off.mean(1, keepdim=True) if kind == "layer" else 0.0
        each = off + shift
        rel = (k / 2 + 10) * F32 + each.square().mean(1, keepdim=True).sqrt() * rstd
        return y + b, (each * rstd * w).abs() + y.abs() * rel + (y.abs() + b.abs() if torch.is_tensor(b) else y.abs()) * 2 * F32

    zero = torch.zeros(1, dtype=torch.float64, device=branch.device)
    x, off = branch.double(), torch.zeros_like(branch, dtype=torch.float64)
    if post:
        x, off = normed(x, post, one("post_weight", zero + 1), one("post_bias", zero), off)
    g = one("gate", zero + 1)
    r = scale * residual.double() + g * x
    off_r = (g * off).abs() + 3 * F32 * ((scale * residual.double()).abs() + (g * x).abs())
    h, off_h = normed(r, norm, one("weight", zero + 1), one("bias", zero), off_r)
    if p["mod_scale"] is not None:
        m = 1 + p["mod_scale"].double()
        off_h = (off_h * m).abs() + 4 * F32 * ((h * m).abs() + p["mod_shift"].double().abs())
        h = h * m + p["mod_shift"].double()
    return r, h, off_r * 1.01 + r.abs() * BF, off_h * 1.01


def _norm_case(m, k, norm, post, vectors, seed, gated=True, modulated=True, affine=True, scale=1.0, by=1.0):
    gen = _gen(seed)
    branch, residual = _randn(gen, m, k, by=0.7 * by), _randn(gen, m, k, at=0.5 * by, by=by)
    shape = (k,) if vectors == 0 else (vectors, k)
    p = {"weight": _randn(gen, k, at=1.0, by=0.1) if affine else None, "bias": _randn(gen, k, by=0.1) if affine and norm == "layer" else None,
         "post_weight": _randn(gen, k, at=1.0, by=0.1) if post and affine else None,
         "post_bias": _randn(gen, k, by=0.1) if post == "layer" and affine else None,
         "gate": _randn(gen, *shape, by=0.5) if gated else None, "mod_scale": _randn(gen, *shape, by=0.2) if modulated else None,
         "mod_shift": _randn(gen, *shape, by=0.2) if modulated else None}
    rows = torch.randint(0, vectors, (m,), generator=gen, device="cuda", dtype=torch.int32) if vectors and (gated or modulated) else None
    each = {n: t if t is None or rows is None or n not in ("gate", "mod_scale", "mod_shift") else t[rows.long()] for n, t in p.items()}
    return branch, residual, p, rows, _norm_reference(branch, residual, each, norm, post, 1e-6, scale)


def _check_norm(got, ref, quantized=True):
    r, h, tol_r, tol_h = ref
    assert got[0].dtype == torch.bfloat16 and float(((got[0].double() - r).abs() - tol_r).max()) <= 0
    if not quantized:
        assert float(((got[1].double() - h).abs() - tol_h - h.abs() * BF * 1.01).max()) <= 0
        return
    q, s = got[1], got[2]
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and s.shape == (r.shape[0], 1)
    top = h.abs().amax(1, keepdim=True)
    want = torch.where(top > 0, top / 448, torch.ones_like(top))
    off = tol_h.amax(1, keepdim=True) / 448 + want * 2 * F32
    assert float(((s.double() - want).abs() - off).max()) <= 0
    # e4m3: 2^-4 of the value, 2^-10 among the subnormal ones; the quotient and its saturation as exact as h and the scale
    exact = h / s.double()
    tol = exact.abs() * 2.0 ** -4 + 2.0 ** -10 + tol_h / s.double() * 1.1 + 448 * 4 * F32
    assert float(((q.double() - exact).abs() - tol).max()) <= 0
    if len(got) == 4:
        assert float(((got[3].double() - h).abs() - tol_h - h.abs() * BF * 1.01).max()) <= 0


@pytest.mark.parametrize("m,k", ((1, 1), (1, 8), (3, 7), (16, 1536), (2, 2048), (5, 1111), (130, 256), (1030, 264), (1500, 2048), (1025, 2047), (40, 6144),
                                 (1100, 4096), (3, 8200), (2, 20000), (1, 32768)))
@pytest.mark.parametrize("norm,post", (("rms", None), ("layer", "layer"), ("rms", "rms"), ("layer", None)))
def test_residual_norm(m, k, norm, post):
    from sacq_b200 import residual_norm_quantize_rows
    branch, residual, p, rows, ref = _norm_case(m, k, norm, post, 0, seed=m + k)
    got = residual_norm_quantize_rows(branch, residual, p["weight"], p["bias"], norm=norm, post_norm=post, post_weight=p["post_weight"],
                                      post_bias=p["post_bias"], gate=p["gate"], mod_scale=p["mod_scale"], mod_shift=p["mod_shift"],
                                      return_normalized=True)
    _check_norm(got, ref)
    plain = residual_norm_quantize_rows(branch, residual, p["weight"], p["bias"], norm=norm, post_norm=post, post_weight=p["post_weight"],
                                        post_bias=p["post_bias"], gate=p["gate"], mod_scale=p["mod_scale"], mod_shift=p["mod_shift"],
                                        quantize=False)
    assert len(plain) == 2 and torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[3])


@pytest.mark.parametrize("m", (1, 19, 2100))
def test_residual_norm_vectors_of_each_request(m):
    from sacq_b200 import residual_norm_quantize_rows
    for gated, modulated in ((True, False), (False, True), (True, True)):
        branch, residual, p, rows, ref = _norm_case(m, 520, "layer", "rms", 5, seed=m, gated=gated, modulated=modulated, scale=0.75)
        got = residual_norm_quantize_rows(branch, residual, p["weight"], p["bias"], norm="layer", post_norm="rms", post_weight=p["post_weight"],
                                          gate=p["gate"], mod_scale=p["mod_scale"], mod_shift=p["mod_shift"], vector_rows=rows, residual_scale=0.75)
        _check_norm(got, ref)
    # a row outside of the table makes its own token NaN and no other
    rows[0], keep = 5, residual_norm_quantize_rows(branch, residual, gate=p["gate"], vector_rows=rows, quantize=False)
    bad = rows.clone()
    bad[m // 2] = -1
    got = residual_norm_quantize_rows(branch, residual, gate=p["gate"], vector_rows=bad, quantize=False)
    clean = torch.ones(m, dtype=torch.bool, device="cuda")
    clean[0] = clean[m // 2] = False
    assert torch.equal(got[0][clean], keep[0][clean]) and bool(got[0][~clean].isnan().all()) and bool(got[1][~clean].isnan().all())


@pytest.mark.parametrize("m,k", ((9001, 8), (3000, 256), (4500, 520), (2500, 768), (2000, 1000), (1800, 1792), (2700, 2048), (1200, 2056), (1100, 8192)))
@pytest.mark.parametrize("vectors", (0, 7))
def test_residual_norm_of_many_rows(m, k, vectors):
    """Each width of the kernels for many rows, several rows after another, with and without tables."""
    from sacq_b200 import residual_norm_quantize_rows
    for norm, post, modulated, affine in (("rms", "rms", False, True), ("rms", None, False, False), ("layer", "layer", True, True)):
        branch, residual, p, rows, ref = _norm_case(m, k, norm, post, vectors, seed=m + k, modulated=modulated, affine=affine)
        got = residual_norm_quantize_rows(branch, residual, p["weight"], p["bias"], norm=norm, post_norm=post, post_weight=p["post_weight"],
                                          post_bias=p["post_bias"], gate=p["gate"], mod_scale=p["mod_scale"], mod_shift=p["mod_shift"],
                                          vector_rows=rows)
        _check_norm(got, ref)


def test_residual_norm_without_vectors_zeros_and_what_is_not_finite():
    from sacq_b200 import residual_norm_quantize_rows
    for m in (4, 1200):
        branch, residual, p, rows, ref = _norm_case(m, 512, "rms", None, 0, seed=m, gated=False, modulated=False, affine=False, scale=0.5, by=30.0)
        _check_norm(residual_norm_quantize_rows(branch, residual, residual_scale=0.5), ref)
        branch[1], residual[1] = 0, 0
        branch[2, 7], residual[3, 9] = INF, NAN
        r, q, s = residual_norm_quantize_rows(branch, residual)
        assert float(s[1]) == 1.0 and bool((q[1].float() == 0).all()) and bool((r[1] == 0).all())
        assert bool(q[3].float().isnan().all()) and float(s[3]) == 1.0
        assert bool(torch.isfinite(q[4:].float()).all()) and bool(q[2, 7].float().isnan())


def test_residual_norm_reads_views_where_they_lie():
    from sacq_b200 import residual_norm_quantize_rows
    gen = _gen(2)
    for m, k, pad in ((33, 512, 8), (1500, 512, 8), (33, 511, 1), (1500, 512, 3)):
        both = _randn(gen, m, 2 * (k + pad))
        branch, residual = both[:, :k], both[:, k + pad:2 * k + pad]
        got = residual_norm_quantize_rows(branch, residual)
        want = residual_norm_quantize_rows(branch.contiguous(), residual.contiguous())
        if pad != 3:                                  # rows that are 16-byte aligned in one of the two only are summed in another order
            assert _same(got, want)
        _check_norm(got, _norm_reference(branch, residual, dict.fromkeys(("weight", "bias", "post_weight", "post_bias", "gate", "mod_scale", "mod_shift")),
                                         "rms", None, 1e-6, 1.0))
        across = residual.t().contiguous().t()
        _check_norm(residual_norm_quantize_rows(branch, across), _norm_reference(branch, residual, dict.fromkeys(
            ("weight", "bias", "post_weight", "post_bias", "gate", "mod_scale", "mod_shift")), "rms", None, 1e-6, 1.0))


# ----------------------------------------------------------------------------- streams and graphs

def _steps(x, inputs):
    """A run of the operators together: norm, rotary, attention, norm."""
    from sacq_b200 import attention_packed, residual_norm_quantize_rows, rotate_heads
    r, h = residual_norm_quantize_rows(x, inputs["residual"], inputs["weight"], quantize=False)
    t = h.view(x.shape[0], 8, 64)
    q, k = rotate_heads(t[:, :4], t[:, 4:6], inputs["positions"], inputs["freq"])
    a = attention_packed(q, k, t[:, 6:], inputs["cu"], causal=True)
    return residual_norm_quantize_rows(torch.cat([a.reshape(x.shape[0], 256)] * 2, 1), r, gate=inputs["weight"], return_normalized=True)


def _steps_inputs(seed, lengths):
    from sacq_b200 import rotary_frequencies
    gen = _gen(seed)
    t = sum(lengths)
    return _randn(gen, t, 512), {"residual": _randn(gen, t, 512), "weight": _randn(gen, 512, at=1.0, by=0.1), "cu": _offsets(lengths),
                                 "positions": torch.cat([torch.arange(n) for n in lengths]).to(torch.int32).cuda(),
                                 "freq": rotary_frequencies(64)[0]}


def _same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def test_steps_together_and_in_graphs():
    x, inputs = _steps_inputs(1, [200, 30, 1, 90])
    want = _steps(x, inputs)
    # the steps one by one in float64, from each step's own bf16 inputs
    from sacq_b200 import attention_packed, residual_norm_quantize_rows, rotate_heads
    none = dict.fromkeys(("weight", "bias", "post_weight", "post_bias", "gate", "mod_scale", "mod_shift"))
    r, h = residual_norm_quantize_rows(x, inputs["residual"], inputs["weight"], quantize=False)
    _check_norm((r, h), _norm_reference(x, inputs["residual"], {**none, "weight": inputs["weight"]}, "rms", None, 1e-6, 1.0), False)
    t = h.view(-1, 8, 64)
    q, k = rotate_heads(t[:, :4], t[:, 4:6], inputs["positions"], inputs["freq"])
    a, lse = attention_packed(q, k, t[:, 6:], inputs["cu"], causal=True, return_lse=True)
    lengths = [200, 30, 1, 90]
    _check_attention(a, lse, _attention_reference(q, k, t[:, 6:], lengths, lengths, True))
    branch = torch.cat([a.reshape(-1, 256)] * 2, 1)
    _check_norm(want, _norm_reference(branch, r, {**none, "gate": inputs["weight"]}, "rms", None, 1e-6, 1.0))
    # two graphs of the same calls, replayed on streams of their own, with other inputs copied in
    graphs = []
    for seed in (2, 3):
        xs, ins = _steps_inputs(seed, [200, 30, 1, 90])
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            _steps(xs, ins)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            made = _steps(xs, ins)
        graphs.append((g, xs, ins, made))
    other = [_steps_inputs(seed, [200, 30, 1, 90]) for seed in (4, 5)]
    wants = [_steps(*o) for o in other]
    for (g, xs, ins, made), (nx, nins) in zip(graphs, other):
        xs.copy_(nx)
        ins["residual"].copy_(nins["residual"])
        ins["weight"].copy_(nins["weight"])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, (g, *_rest) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(_same(made, w) for (_, _, _, made), w in zip(graphs, wants))


def test_attention_split_over_keys_in_graphs_on_two_streams():
    """A long past is worked on in parts whose results are joined: each call has its own room for them."""
    from sacq_b200 import attention_packed
    sets = []
    for seed in range(4):
        gen = _gen(seed)
        q, k, v = _randn(gen, 2, 4, 128), _randn(gen, 9000, 2, 128), _randn(gen, 9000, 2, 128)
        sets.append((q, k, v, _offsets([1, 1]), _offsets([7000, 2000])))
    want = [attention_packed(*s, causal=True) for s in sets]
    for s, w in zip(sets, want):
        ref = _attention_reference(*s[:3], [1, 1], [7000, 2000], True)
        assert float(((w.double() - ref[0]).abs() - ref[2]).max()) <= 0
    streams = [torch.cuda.Stream() for _ in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attention_packed(*s, causal=True))
        graphs.append(g)
    for _ in range(5):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                eager.append(attention_packed(*s, causal=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(outs, want)) and all(torch.equal(a, w) for a, w in zip(eager, want))


def test_steps_follow_the_kernel_in_front():
    """Each step is launched early behind its predecessor and reads nothing before that one has finished."""
    x, inputs = _steps_inputs(6, [150, 90])
    want = _steps(x.clone() * 0.5, inputs)
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        y = x * 0
        for _ in range(3):
            big = big @ big * 1e-3
        y.add_(x, alpha=0.5)
        assert _same(_steps(y, inputs), want)


def test_policy_of_prompts_of_different_lengths():
    """The packed forward gives each request what it gets alone, up to the roundings that other kernels of the linears bring
    (the bar of the batched policy: 2e-2 relative), and requests do not reach each other."""
    from sacq_b200.policy import SyntheticGr00tPolicy
    policy = SyntheticGr00tPolicy("cuda", seed=3)
    image, noise = policy.example_inputs(9, batch=3)
    lengths = [44, 0, 17]
    got = policy.forward_packed(image, noise, lengths)
    assert tuple(got.shape) == (3, 16, 32) and bool(torch.isfinite(got.float()).all())
    assert torch.equal(got, policy.forward_packed(image, noise, lengths))
    for i in range(3):
        one = policy.forward_packed(image[i:i + 1], noise[i:i + 1], lengths[i:i + 1])[0]
        err = ((got[i].float() - one.float()).norm() / one.float().norm()).item()
        assert err <= 2e-2, (i, err)
    other = image.clone()
    other[1] = 1.0 - other[1]
    again = policy.forward_packed(other, noise, lengths)
    assert torch.equal(again[0], got[0]) and torch.equal(again[2], got[2]) and not torch.equal(again[1], got[1])
    for bad in ([44, 0], [44, 0, 45], [-1, 0, 1]):
        with pytest.raises(ValueError):
            policy.forward_packed(image, noise, bad)


def test_rotary_results_lie_in_one_buffer_of_any_order():
    from sacq_b200 import rotary_frequencies, rotate_heads
    gen = torch.Generator(device="cuda").manual_seed(21)
    t, h, d = 37, 3, 64
    q, k = _randn(gen, t, h, d), _randn(gen, t, h, d)
    pos, (freq, _) = torch.arange(t, device="cuda"), rotary_frequencies(d)
    want = rotate_heads(q, k, pos, freq)
    for views in (lambda x: (x[:, :h], x[:, h:]), lambda x: (x[:, ::2], x[:, 1::2])):
        made = torch.zeros(t, 2 * h, d, device="cuda", dtype=torch.bfloat16)
        rotate_heads(q, k, pos, freq, out=views(made))
        turned = torch.zeros_like(made)
        views(turned)[0].copy_(q)
        views(turned)[1].copy_(k)
        rotate_heads(*views(turned), pos, freq, out=views(turned))
        for x in (made, turned):
            assert all(torch.equal(a, b) for a, b in zip(views(x), want))
    assert all(torch.equal(a, b) for a, b in zip(rotate_heads(q, q, pos, freq), (want[0], want[0])))


def test_steps_refuse_what_they_cannot_do():
    from sacq_b200 import attention_packed, residual_norm_quantize_rows, rotary_frequencies, rotate_heads
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, k, cu = z(4, 4, 64), z(4, 2, 64), _offsets([4])
    for args in ((q, k, z(5, 2, 64), cu), (q, z(4, 3, 64), z(4, 3, 64), cu), (q, z(4, 2, 32), z(4, 2, 32), cu), (z(4, 4, 264), z(4, 2, 264), z(4, 2, 264), cu),
                 (q, k, k, cu, _offsets([2, 2])), (q, k, k, cu.cpu())):
        with pytest.raises(ValueError):
            attention_packed(*args)
    for args in ((q, k, k, cu.long()), (q, k, k, cu.view(1, -1)), (q.float(), k, k, cu)):
        with pytest.raises(TypeError):
            attention_packed(*args)
    for scale in (0.0, -1.0, INF, NAN):
        with pytest.raises(ValueError):
            attention_packed(q, k, k, cu, scale=scale)
    for out in (q, z(4, 4, 32), z(4, 64, 4).transpose(1, 2), z(3, 4, 64), z(1, 4, 64).expand(4, 4, 64)):
        with pytest.raises(ValueError):
            attention_packed(q, k, k, cu, out=out)
    grad = z(4, 4, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        attention_packed(grad, k, k, cu)
    with torch.no_grad():
        attention_packed(grad, k, k, cu)
    pos, (freq, _) = torch.zeros(4, dtype=torch.int32, device="cuda"), rotary_frequencies(64)
    for args in ((q, z(5, 2, 64), pos, freq), (q, k, pos[:3], freq), (q, k, pos, torch.cat([freq, freq])), (q, k, pos.cpu(), freq), (q, k, pos, freq[:0])):
        with pytest.raises(ValueError):
            rotate_heads(*args)
    for args in ((q, k, pos.float(), freq), (q, k, pos, freq.float())):
        with pytest.raises(TypeError):
            rotate_heads(*args)
    whole = z(5, 4, 64)
    with pytest.raises(ValueError, match="overlaps"):
        rotate_heads(whole[:4], None, pos, freq, out=(whole[1:], None))
    two = z(4, 4, 64)
    for out in ((two, q), (two, two), (two, None), (None, q), (z(1, 4, 64).expand(4, 4, 64), None)):
        with pytest.raises(ValueError):
            rotate_heads(q, two, pos, freq, out=out)
    for out in ((q, None), (None, q), (q, q)):                    # the same heads twice, one of them turned in place
        with pytest.raises(ValueError, match="overlap"):
            rotate_heads(q, q, pos, freq, out=out)
    with pytest.raises(RuntimeError, match="no_grad"):
        rotate_heads(grad, k, pos, freq)
    x, v = z(4, 64), z(64)
    rows = torch.zeros(4, dtype=torch.int32, device="cuda")
    for kw in (dict(post_weight=v), dict(mod_scale=v), dict(gate=z(65)), dict(weight=z(63)), dict(eps=-1.0), dict(vector_rows=rows), dict(gate=v, vector_rows=rows),
               dict(gate=z(2, 64), mod_scale=z(3, 64), mod_shift=z(3, 64), vector_rows=rows), dict(gate=z(2, 64), vector_rows=rows[:3])):
        with pytest.raises(ValueError):
            residual_norm_quantize_rows(x, x, **kw)
    for kw in (dict(weight=v.float()), dict(gate=v.cpu()), dict(gate=z(2, 64), vector_rows=rows.long())):
        with pytest.raises(TypeError):
            residual_norm_quantize_rows(x, x, **kw)
    with pytest.raises(ValueError):
        residual_norm_quantize_rows(x, z(3, 64))
    empty = residual_norm_quantize_rows(z(0, 64), z(0, 64))
    assert [t.shape for t in empty] == [(0, 64), (0, 64), (0, 1)]


def test_the_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    code = """
import torch
from sacq_b200 import attention_packed, residual_norm_quantize_rows, rotary_frequencies, rotate_heads
g = torch.Generator(device="cuda").manual_seed(0)
r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
q, k, v, x, y = r(3000, 4, 64), r(3000, 2, 64), r(3000, 2, 64), r(3000, 256), r(3000, 256)
cu = torch.tensor([0, 1000, 3000], dtype=torch.int32, device="cuda")
one = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
pos, (freq, _) = torch.arange(3000, device="cuda"), rotary_frequencies(64)
def calls():
    a, b = rotate_heads(q, k, pos, freq)
    return [a, b, attention_packed(a, b, v, cu, causal=True), attention_packed(q[:2], k, v, one, cu), *residual_norm_quantize_rows(x, y)[::2]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    made = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(m, e) for m, e in zip(made, calls()))
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


def _cut_up(q, k, v, cu_q, cu_k, causal=False):
    """Whether the call's keys go in chunks: it needs room for their results."""
    import ctypes
    from sacq_b200 import _lib
    d = _lib.AttentionDesc(struct_size=ctypes.sizeof(_lib.AttentionDesc), causal=causal, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=q.data_ptr(),
                           tokens_q=q.shape[0], tokens_k=k.shape[0], cu_q=cu_q.data_ptr(), cu_k=cu_k.data_ptr(), sequences=cu_q.numel() - 1,
                           heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2], scale=1.0)
    for n, t in (("q", q), ("k", k), ("v", v), ("out", q)):
        setattr(d, n + "_token", t.stride(0))
        setattr(d, n + "_head", t.stride(1))
    return _lib.load().sacq_attention_workspace_bytes(ctypes.byref(d)) > 0


@pytest.mark.parametrize("cu_q,cu_k,heads,kv_heads,dim,cut", (
    ([0, 1, 2, 0, 0, 0, 0, 0, 0], [0, 9000, 18000, 0, 0, 0, 0, 0, 0], 4, 2, 128, True),                  # 16-row tiles
    ([0, 100, 200, 0, 0, 0, 0, 0, 0], [0, 9000, 18000, 0, 0, 0, 0, 0, 0], 4, 2, 64, True),               # 128-row tiles
    ([40, 60, 20, 30, 0, 15], [2000, 9000, 1000, 2000, 0, 1000], 2, 2, 64, True),
    ([40, 60, 20, 30, 0, 15], [2000, 9000, 1000, 2000, 0, 1000], 8, 1, 128, True),
    ([0, 10, 50, 0, 0, 0, 0, 0], [0, 10, 50, 0, 0, 0, 0, 0], 2, 1, 36, False),                           # a warp per row
    ([40, 60, 20, 30, 0, 15], [200, 900, 100, 200, 0, 100], 2, 1, 36, False),
    ([0, 10, 50, 0, 0, 0, 0, 0], [0, 10, 50, 0, 0, 0, 0, 0], 2, 1, 64, False),
    ([0] * 70 + [3, 8] + [0] * 70, [0] * 70 + [40, 60] + [0] * 70, 2, 1, 36, False)))
@pytest.mark.parametrize("causal", (False, True))
def test_attention_of_offsets_that_go_down(cu_q, cu_k, heads, kv_heads, dim, cut, causal):
    """Sequences in any order, empty ones anywhere: each row of a sequence is made by every kernel, and no other row is touched."""
    from sacq_b200 import attention_packed
    gen = _gen(11)
    spans = [(a, max(b - a, 0), c, max(d - c, 0)) for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:])]
    tokens_q, tokens_k = max(cu_q) + 5, max(cu_k) + 5
    q = _randn(gen, tokens_q, heads, dim, by=1.5)
    k, v = (_randn(gen, tokens_k, kv_heads, dim, by=1.5) for _ in range(2))
    offsets = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cu_q, cu_k)]
    assert _cut_up(q, k, v, *offsets, causal) == cut
    out = torch.full_like(q, 3.0)
    lse = attention_packed(q, k, v, *offsets, causal=causal, out=out, return_lse=True)[1]
    left = torch.ones(tokens_q, dtype=torch.bool, device="cuda")
    for at_q, nq, at_k, nk in spans:
        if nq == 0:
            continue
        rows, keys = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
        _check_attention(out[rows], lse[rows], _attention_reference(q[rows], k[keys], v[keys], [nq], [nk], causal))
        left[rows] = False
    assert bool((out[left] == 3).all())


@pytest.mark.parametrize("lq,past,heads,kv_heads,dim", ((32, 0, 1, 1, 64), (27, 0, 2, 2, 128), (17, 0, 1, 1, 40), (16, 8, 2, 1, 128), (16, 30, 4, 2, 64), (9, 23, 3, 1, 96),
                                                        (3, 0, 2, 1, 64), (16, 7001, 2, 1, 128), (30, 9020, 1, 1, 64), (16, 90, 2, 1, 72)))
@pytest.mark.parametrize("value", (NAN, INF))
def test_attention_of_few_queries_keeps_later_keys_out(value, lq, past, heads, kv_heads, dim):
    """16-row tiles: for every token, all keys behind those that it sees hold anything."""
    from sacq_b200 import attention_packed
    gen = _gen(12)
    n = past + lq
    q, k, v = _randn(gen, lq, heads, dim), _randn(gen, n, kv_heads, dim), _randn(gen, n, kv_heads, dim)
    cu_q, cu_k = _offsets([lq]), _offsets([n])
    assert lq * (heads // kv_heads) <= 32 and _cut_up(q, k, v, cu_q, cu_k, True) == (past > 5000)
    ref = _attention_reference(q, k, v, [lq], [n], True)
    for t in range(lq):
        k2, v2 = k.clone(), v.clone()
        k2[past + t + 1:], v2[past + t + 1:] = value, value
        got, lse = attention_packed(q, k2, v2, cu_q, cu_k, causal=True, return_lse=True)
        _check_attention(got[:t + 1], lse[:t + 1], tuple(x[:t + 1] for x in ref))


@pytest.mark.parametrize("lq,lk", (([5, 16, 2], [37, 70, 61]), ([1, 1, 1], [200, 16, 33]), ([4, 9, 1], [9000, 7, 50])))
@pytest.mark.parametrize("heads,kv_heads,dim", ((2, 1, 128), (2, 2, 64), (3, 1, 24)))
@pytest.mark.parametrize("value", (NAN, -INF))
def test_attention_of_few_queries_keeps_other_sequences_out(value, heads, kv_heads, dim, lq, lk):
    from sacq_b200 import attention_packed
    gen = _gen(13)
    q = _randn(gen, sum(lq) + 6, heads, dim)
    k, v = (_randn(gen, sum(lk) + 6, kv_heads, dim) for _ in range(2))
    cu_q, cu_k = _offsets(lq) + 3, _offsets(lk) + 3
    at_q = at_k = 3
    for nq, nk in zip(lq, lk):
        rows, keys = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
        others = [torch.full_like(t, value) for t in (q, k, v)]
        for o, t, s in zip(others, (q, k, v), (rows, keys, keys)):
            o[s] = t[s]
        for causal in (False, True):
            got, lse = attention_packed(*others, cu_q.to(torch.int32), cu_k.to(torch.int32), causal=causal, return_lse=True)
            _check_attention(got[rows], lse[rows], _attention_reference(q[rows], k[keys], v[keys], [nq], [nk], causal))
        at_q, at_k = at_q + nq, at_k + nk


@pytest.mark.parametrize("lq,heads,kv_heads,dim,cut", ((3, 4, 2, 128, True), (1, 1, 1, 64, True), (100, 4, 4, 128, True), (100, 4, 4, 64, True), (100, 16, 16, 64, False),
                                                       (70, 2, 1, 36, False)))
def test_attention_of_keys_that_score_minus_infinity(lq, heads, kv_heads, dim, cut):
    """Keys whose scores are -inf have no weight, also where a whole chunk has no others; a row with no other key is NaN, as in the formula."""
    from sacq_b200 import attention_packed
    gen = _gen(14)
    lk = 4100 if cut else 300
    none = lk // 4 * 3
    q = _randn(gen, lq, heads, dim).abs() + 0.125
    k, v = (_randn(gen, lk, kv_heads, dim) for _ in range(2))
    k[:none] = -INF
    cu_q, cu_k = _offsets([lq]), _offsets([lk])
    assert _cut_up(q, k, v, cu_q, cu_k) == cut
    got, lse = attention_packed(q, k, v, cu_q, cu_k, return_lse=True)
    _check_attention(got, lse, _attention_reference(q, k[none:], v[none:], [lq], [lk - none], False))
    k[none:] = -INF
    got, lse = attention_packed(q, k, v, cu_q, cu_k, return_lse=True)
    assert bool(got.isnan().all()) and bool((lse == -INF).all() or lse.isnan().all())
    v[5] = INF                               # a weight of zero times infinity: NaN, in whichever chunk it is
    k[none:] = 0.0
    got = attention_packed(q, k, v, cu_q, cu_k)
    assert bool(got[:, :heads // kv_heads].isnan().all())


@pytest.mark.parametrize("lq,lk,heads,kv_heads", (([40, 90], [700, 300], 2, 2), ([140, 3], [900, 140], 4, 2), ([40, 90], [9000, 300], 2, 2)))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("factor", (NAN, 100.0))
def test_attention_of_a_request_does_not_depend_on_its_neighbours_values(factor, dim, lq, lk, heads, kv_heads):
    """To the bit: its neighbours' queries lie in the same tile."""
    from sacq_b200 import attention_packed
    gen = _gen(15)
    q = _randn(gen, sum(lq), heads, dim)
    k, v = (_randn(gen, sum(lk), kv_heads, dim) for _ in range(2))
    cu_q, cu_k = _offsets(lq), _offsets(lk)
    want = attention_packed(q, k, v, cu_q, cu_k, return_lse=True)
    q[lq[0]:] *= factor
    v[lk[0]:] *= factor
    k[lk[0]:] *= factor
    got = attention_packed(q, k, v, cu_q, cu_k, return_lse=True)
    assert all(torch.equal(g[:lq[0]], w[:lq[0]]) for g, w in zip(got, want))


@pytest.mark.parametrize("m,k", ((40, 64), (1500, 520), (1100, 2048), (1100, 2056), (1030, 1111), (20, 6144)))
def test_residual_norm_makes_8_bit_rows_as_the_quantizer_does(m, k):
    """Rows that are their own shift to the bit, of maxima of any size, against quantize_rows: the same scales and bytes."""
    from sacq_b200 import quantize_rows, residual_norm_quantize_rows
    gen = _gen(m + k)
    shift = _randn(gen, m, k, by=1.0) * (torch.randint(-40, 40, (m, 1), generator=gen, device="cuda").float().exp2()).to(torch.bfloat16)
    rows = torch.randperm(m, generator=gen, device="cuda").to(torch.int32)
    zero = torch.zeros(k, dtype=torch.bfloat16, device="cuda")
    _, q, s = residual_norm_quantize_rows(_randn(gen, m, k), _randn(gen, m, k), zero, mod_scale=torch.zeros_like(shift), mod_shift=shift, vector_rows=rows)
    want_q, want_s = quantize_rows(shift[rows.long()])
    assert torch.equal(s.view(-1), want_s.view(-1))
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


def test_steps_refuse_forward_mode_tangents():
    import torch.autograd.forward_ad as forward_ad
    from sacq_b200 import attention_packed, residual_norm_quantize_rows, rotary_frequencies, rotate_heads
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, k, cu = z(4, 4, 64), z(4, 2, 64), _offsets([4])
    pos, (freq, _) = torch.zeros(4, dtype=torch.int32, device="cuda"), rotary_frequencies(64)
    x, v = z(4, 64), z(64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: attention_packed(dual(q), k, k, cu), lambda: attention_packed(q, k, dual(k), cu), lambda: attention_packed(q, k, k, cu, out=dual(z(4, 4, 64))),
                     lambda: rotate_heads(dual(q), k, pos, freq), lambda: rotate_heads(q, dual(k), pos, freq),
                     lambda: residual_norm_quantize_rows(dual(x), x), lambda: residual_norm_quantize_rows(x, dual(x)),
                     lambda: residual_norm_quantize_rows(x, x, dual(v)), lambda: residual_norm_quantize_rows(x, x, gate=dual(v))):
            with pytest.raises(RuntimeError, match="derivative"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="derivative"):
                call()
        attention_packed(forward_ad.unpack_dual(dual(q)).primal, k, k, cu)


def test_the_status_of_bounded_waits_is_read_per_device():
    from sacq_b200 import block_steps_status
    assert block_steps_status() == 0 and block_steps_status("cuda:0") == 0 and block_steps_status(torch.device("cuda", 0)) == 0
    with pytest.raises((RuntimeError, AssertionError)):
        block_steps_status(torch.cuda.device_count())


def _fastest(call):
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("lengths,past,heads,kv_heads", (([5000], 0, 4, 4), ([16] * 300, 400, 4, 2)))
@pytest.mark.parametrize("dim", (64, 128))
def test_attention_of_infinities_that_are_seen_makes_no_row_again(lengths, past, heads, kv_heads, dim):
    """What a row sees is in its result at once.  (Rows made again one by one took 100 to 250 times as long as the call.)"""
    from sacq_b200 import attention_packed
    gen = _gen(16)
    lk = [past + n for n in lengths]
    q = _randn(gen, sum(lengths), heads, dim)
    k, v = (_randn(gen, sum(lk), kv_heads, dim) for _ in range(2))
    cu_q, cu_k = _offsets(lengths), _offsets(lk)
    call = lambda: attention_packed(q, k, v, cu_q, cu_k, causal=True)  # noqa: E731
    clean = call()
    plain = _fastest(call)
    v[cu_k[:-1].long(), :, 3] = NAN
    got = call()
    assert bool(got[..., 3].isnan().all()) and torch.equal(got[..., :3], clean[..., :3]) and torch.equal(got[..., 4:], clean[..., 4:])
    assert _fastest(call) <= 4 * plain


@pytest.mark.parametrize("heads,kv_heads,dim", ((16, 8, 128), (16, 16, 64), (8, 1, 96), (24, 24, 32)))
@pytest.mark.parametrize("causal", (False, True))
def test_attention_of_more_items_than_the_device_has_room_for(heads, kv_heads, dim, causal):
    """128-row tiles: CTAs take item after item, of one to nine steps of keys, lone tiles and pairs, and items that have not begun."""
    lengths = [57 + (41 * i) % 244 for i in range(40)]
    for at, n in ((3, 1), (7, 0), (11, 9), (20, 1100), (33, 700)):
        lengths[at] = n
    _attend(lengths, lengths, heads, kv_heads, dim, causal, seed=17)
    others = [lengths[(7 * i + 5) % 40] for i in range(40)]
    _attend(lengths, others, heads, kv_heads, dim, causal, seed=18)


@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("causal", (False, True))
def test_attention_of_more_chunks_than_the_device_has_room_for(dim, causal):
    lq, lk = [80] * 8, [16000] + [100 + 33 * i for i in range(7)]
    z = lambda t, h: torch.empty(t, h, dim, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    assert _cut_up(z(sum(lq), 8), z(sum(lk), 8), z(sum(lk), 8), _offsets(lq), _offsets(lk), causal)
    _attend(lq, lk, 8, 8, dim, causal, seed=19)


@pytest.mark.parametrize("dim", (64, 128))
def test_attention_of_few_queries_of_more_items_than_the_device_has_room_for(dim):
    lq, lk = [1 + i % 16 for i in range(90)], [(97 * i) % 700 for i in range(90)]
    for causal in (False, True):
        _attend(lq, lk, 16, 8, dim, causal, seed=20)


def _block_reference(blk, x, lengths, causal=False, rotary=None, cross=None, modulation=None, gates=(None, None)):
    """A block on packed rows from its own quantized linears, one at a time, and float64 norms, rotation and attention: what
    _Block.forward states for each sequence, with gates on the attention branches."""
    from sacq_b200 import act_quantize_rows, quantize_rows
    bf = torch.bfloat16
    t = x.shape[0]
    zero = torch.zeros(blk.hidden, dtype=bf, device=x.device)
    m = (zero,) * 4 if modulation is None else modulation.view(4, blk.hidden)         # shift, scale in front of attention; the same in front of the MLP

    def rows(norm, x, shift, scale):
        h = torch.nn.functional.layer_norm(x.double(), (blk.hidden,), None if norm.weight is None else norm.weight.double(),
                                           None if norm.bias is None else norm.bias.double(), norm.eps)
        return quantize_rows((h * (1 + scale.double()) + shift.double()).to(bf))

    def attend(q, k, v, lq, lk, causal):
        heads = lambda y: y.view(y.shape[0], -1, blk.head_dim)  # noqa: E731
        return _attention_reference(heads(q), heads(k), heads(v), lq, lk, causal)[0].to(bf).view(t, blk.hidden)

    def add(x, branch, gate):
        return (x.double() + (1.0 if gate is None else gate.double()) * branch.double()).to(bf)

    q, k, v = (layer.linear_a8(*rows(blk.n1, x, m[0], m[1])) for layer in (blk.q, blk.k, blk.v))
    if rotary is not None:
        q, k = (_rotary_reference(y.view(t, -1, blk.head_dim), *rotary, "half", 1.0)[0].to(bf).view(t, -1) for y in (q, k))
    x = add(x, blk.o(attend(q, k, v, lengths, lengths, causal)), gates[0])
    if cross is not None:
        keys, values, others = cross
        x = add(x, blk.co(attend(blk.cq.linear_a8(*rows(blk.n3, x, zero, zero)), keys, values, lengths, others, False)), gates[1])
    up = blk.up.linear_a8(*rows(blk.n2, x, m[2], m[3]))
    if blk.gated:
        down = act_quantize_rows("silu_mul", blk.gate.linear_a8(*rows(blk.n2, x, m[2], m[3])), up)
    else:
        down = act_quantize_rows("gelu", up)
    return blk.down.linear_a8(*down, residual=x)


@pytest.mark.parametrize("kind", ("vision", "language", "action"))
def test_packed_blocks_against_their_formula(kind):
    """Each kind of block of the packed forward.  Rows that are rounded to bf16 at other places differ by 2^-10 on average, so one e4m3 value in 2^-10 / 2^-3.5
    of its neighbour's distance becomes its neighbour: 2^-6.75 of the norm of what a linear gets, 0.023 after the six that follow
    one another; 0.05 of what the block adds.  The same formula with a gate, a norm's vectors, the rotation, the mask or the context of another place is
    off by twice that at least (the norm in front of the language model's attention has large weights: its scores would be too flat to tell)."""
    from sacq_b200 import rotary_frequencies
    from sacq_b200.policy import _Block, _Factory
    gen = _gen(22)
    f = _Factory(torch.device("cuda"), 5)
    lengths = [70, 1, 33]
    t, hidden = sum(lengths), 512
    x = _randn(gen, t, hidden)
    cu = _offsets(lengths)
    given, wrong, packed = {}, [], {}
    if kind == "vision":
        blk = _Block(f, hidden, 8, 8, 1024, gated=False)
        wrong = [{"lengths": [t]}]
    elif kind == "language":
        blk = _Block(f, hidden, 4, 2, 1024, gated=True)
        positions = torch.cat([torch.arange(n) for n in lengths]).to(torch.int32).cuda()
        given = {"causal": True, "rotary": (positions, rotary_frequencies(128, base=1e6)[0])}
        packed = given
        wrong = [{"causal": False}, {"rotary": None}, {"rotary": (positions * 2, given["rotary"][1])}]
    else:
        blk = _Block(f, hidden, 4, 4, 1024, gated=False, cross_dim=hidden, adaln=True)
        blk.cv = _Factory(torch.device("cuda"), 6).linear(hidden, hidden)             # layers of one shape and factory have one payload
        others = [20, 41, 7]
        context = blk.cross_kv(_randn(gen, sum(others), hidden))
        modulation, gates = _randn(gen, 4 * hidden, by=0.5), _randn(gen, 2, hidden)
        given = {"cross": (*context, others), "modulation": modulation, "gates": gates}
        packed = {"cross": (*context, _offsets(others)), "modulation": modulation, "gates": gates}
        wrong = [{"gates": gates.flip(0)}, {"gates": (None, None)}, {"modulation": modulation.view(4, hidden)[[1, 0, 2, 3]]}, {"modulation": modulation.view(4, hidden)[[2, 3, 0, 1]]},
                 {"cross": (context[1], context[0], others)}, {"cross": (*context, others[::-1])}]
    for norm in (blk.n1, blk.n2, getattr(blk, "n3", None)):
        if norm is not None and norm.weight is not None:
            norm.weight.data.copy_(_randn(gen, hidden, at=2.5 if kind == "language" and norm is blk.n1 else 1.0, by=0.2))
            norm.bias.data.copy_(_randn(gen, hidden, by=0.2))
    with torch.no_grad():
        got = blk.forward_packed(x, cu, **packed)
        ref = _block_reference(blk, x, **{"lengths": lengths, **given})
        added = (ref.double() - x.double()).norm()
        off = lambda y: float((y.double() - ref.double()).norm() / added)  # noqa: E731
        assert off(got) <= 0.05, off(got)
        for w in wrong:
            other = off(_block_reference(blk, x, **{"lengths": lengths, **given, **w}))
            assert other > 0.1, (list(w), other)


def _tail(gen, tokens, last, heads, dim):
    """[tokens, heads, dim] of which the last rows are made; more than 2^31 elements."""
    x = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    x[-last:] = _randn(gen, last, heads, dim)
    return x


@pytest.mark.parametrize("lq,heads,dim", ((200, 16, 128), (5, 16, 128), (20, 16, 40), (20, 16, 36)))
def test_attention_of_keys_behind_two_to_the_31_elements(lq, heads, dim):
    from sacq_b200 import attention_packed
    gen = _gen(23)
    tokens, last = 2_100_003, 700
    q = _randn(gen, lq, heads, dim)
    k, v = (_tail(gen, tokens, last, 8, 128)[..., :dim] for _ in range(2))
    cu_k = torch.tensor([tokens - last, tokens], dtype=torch.int32, device="cuda")
    got, lse = attention_packed(q, k, v, _offsets([lq]), cu_k, causal=True, return_lse=True)
    _check_attention(got, lse, _attention_reference(q, k[-last:], v[-last:], [lq], [last], True))
    # queries and results as far out, the last of their keys with values of no use
    v[-1] = NAN
    far = _tail(gen, 1_100_000, lq, heads, 128)
    far[-lq:, :, :dim] = q
    out = torch.empty_like(far)[..., :dim]
    cu_q = torch.tensor([far.shape[0] - lq, far.shape[0]], dtype=torch.int32, device="cuda")
    got, lse = attention_packed(far[..., :dim], k, v, cu_q, cu_k, causal=True, out=out, return_lse=True)
    _check_attention(got[-lq:-1], lse[-lq:-1], tuple(x[:-1] for x in _attention_reference(q, k[-last:], v[-last:].nan_to_num(0.0), [lq], [last], True)))
    assert bool(got[-1].isnan().all())


def test_rotary_and_norms_behind_two_to_the_31_elements():
    from sacq_b200 import residual_norm_quantize_rows, rotary_frequencies, rotate_heads
    gen = _gen(24)
    tokens, last = 1_050_000, 1500
    q = _tail(gen, tokens, last, 16, 128)
    pos, (freq, _) = torch.arange(tokens, device="cuda"), rotary_frequencies(128)
    for layout, part in (("half", slice(0, 128)), ("interleaved", slice(0, 128)), ("half", slice(1, 128))):
        f = freq if part.start == 0 else rotary_frequencies(40)[0]
        want = rotate_heads(q[-last:, :, part], None, pos[-last:], f, layout=layout)[0]
        assert torch.equal(rotate_heads(q[..., part], None, pos, f, layout=layout)[0][-last:], want)
    x = q.view(tokens, 2048)
    gate = _randn(gen, 3, 2048)
    rows = (torch.arange(tokens, device="cuda") % 3).to(torch.int32)
    kw = lambda s: dict(gate=gate, vector_rows=rows[s], return_normalized=True)  # noqa: E731
    got = residual_norm_quantize_rows(x, x, **kw(slice(None)))
    assert _same([t[-last:] for t in got], residual_norm_quantize_rows(x[-last:], x[-last:], **kw(slice(tokens - last, None))))
    del got
    odd = x[:, :2047]                        # rows that are 16-byte aligned and of odd length: elements one by one
    got = residual_norm_quantize_rows(odd, odd, quantize=False)
    assert _same([t[-last:] for t in got], residual_norm_quantize_rows(odd[-last:], odd[-last:], quantize=False))
    few = x.view(-1, 8192)                   # wide rows
    got = residual_norm_quantize_rows(few, few)
    assert _same([t[-last // 4:] for t in got], [t[-last // 4:] for t in residual_norm_quantize_rows(few[-1100:], few[-1100:])])


@pytest.mark.parametrize("heads,kv_heads,dim,new", ((16, 8, 128, 1), (4, 4, 64, 40), (2, 1, 36, 3)))
def test_attention_of_a_cache_with_room_behind_each_past(heads, kv_heads, dim, new):
    """The room is a sequence without queries, and may hold anything."""
    from sacq_b200 import attention_packed
    gen = _gen(25)
    room, pasts = 4096, [500, 600, 4096, 41]
    q = _randn(gen, new * len(pasts), heads, dim)
    cache = [torch.full((room * len(pasts), kv_heads, dim), NAN, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    rows = torch.cat([torch.arange(n) + i * room for i, n in enumerate(pasts)]).cuda()
    for t in cache:
        t[rows] = _randn(gen, sum(pasts), kv_heads, dim)
    cu_q, cu_k = _offsets([n for _ in pasts for n in (new, 0)]), _offsets([n for past in pasts for n in (past, room - past)])
    got, lse = attention_packed(q, *cache, cu_q, cu_k, causal=True, return_lse=True)
    _check_attention(got, lse, _attention_reference(q, *(t[rows] for t in cache), [new] * len(pasts), pasts, True))


def test_no_wait_has_run_out():
    import ctypes
    from sacq_b200 import _lib
    word = ctypes.c_int(-1)
    _lib.check(_lib.load().sacq_block_steps_status(ctypes.byref(word)))
    assert word.value == 0
