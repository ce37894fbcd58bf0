"""The steps of a transformer block between its quantized projections, as cases that can be timed and compared.

Three operators: attention over packed sequences of different lengths, rotary positions of query and key heads, and the
norms behind and before a block with its gate, its residual scale and the 8-bit rows of the projections that follow.

Heads and widths are those of the synthetic policy (language model 16 query / 8 key-value heads of 128, hidden 2048; vision
tower 16 heads of 64, hidden 1024; action head 12 heads of 128, hidden 1536, 16 steps, 300 language tokens) and generic ones.
A case is a dict: `op` names the operator, the rest its sizes.  `run` computes the operators from elementary tensor
operations in 32 bits, or, where `own` is true, calls the package."""
import math
import random

import torch

own = False

DEVICE = "cuda:0"


# ----------------------------------------------------------------------------- cases

def _attention(name, kind, batch, q_lo, q_hi, k_lo, k_hi, heads, kv_heads, dim, fused=False):
    """kind: "causal" and "full" attend to their own tokens (k_lo and k_hi mean nothing), "cross" to all keys of another length,
    "tail" to a longer past that ends with them.  fused: heads are views of one projection's rows."""
    return {"name": name, "op": "attention", "kind": kind, "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "k_lo": k_lo, "k_hi": k_hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "fused": fused}


def _rotary(name, tokens, heads, kv_heads, dim, rotary_dim, layout, most_position, factor=1.0, fused=False):
    """factor: by how much the context was stretched beyond what the frequencies were made for (1: not at all)."""
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary_dim": rotary_dim, "layout": layout, "most_position": most_position, "factor": factor, "fused": fused}


def _norm(name, m, k, norm, post, gate_rows, modulated, residual_scale=1.0, quantize=True):
    """post: whether the block's output is normed too; gate_rows: 0 for no gate, 1 for one vector, else one for each
    request; modulated: scale and shift vectors behind the second norm, as many as gates."""
    return {"name": name, "op": "norm", "m": m, "k": k, "norm": norm, "post": post, "gate_rows": gate_rows,
            "modulated": modulated, "residual_scale": residual_scale, "quantize": quantize}


def listed():
    return [
        # one control request's action head attending to its own 16 steps: nothing but latency
        _attention("action_self_16", "full", 1, 16, 16, 0, 0, 12, 12, 128),
        # the same head's cross-attention for 64 requests whose prompts differ in length
        _attention("action_cross_b64", "cross", 64, 16, 16, 270, 300, 12, 12, 128),
        # the vision tower on 64 images of 256 patches, heads cut out of one projection's rows
        _attention("vision_b64", "full", 64, 256, 256, 0, 0, 16, 16, 64, fused=True),
        # prefill of 64 prompts of different lengths, grouped heads
        _attention("prefill_ragged_b64", "causal", 64, 57, 300, 0, 0, 16, 8, 128),
        # two long prompts
        _attention("prompt_long", "causal", 2, 6001, 8192, 0, 0, 16, 8, 128),
        # single tokens of 16 conversations against their pasts
        _attention("token_b16", "tail", 16, 1, 1, 501, 16384, 16, 8, 128),
        # positions of a decode batch, far into the conversations
        _rotary("rotary_token_b16", 16, 16, 8, 128, 128, "half", 131072),
        # positions of a batch of prompts, heads cut out of one projection's rows
        _rotary("rotary_prefill", 12001, 16, 8, 128, 128, "half", 300, fused=True),
        # neighbouring pairs of the first half of each head, context stretched sixteenfold
        _rotary("rotary_part_long", 32768, 16, 8, 128, 64, "interleaved", 1000000, factor=16.0),
        # the action head between two projections: gate, residual, modulated LayerNorm, 8-bit rows
        _norm("norm_action_16", 16, 1536, "layer", False, 1, True),
        # an odd width without 8-bit rows: both norms, a residual scale
        _norm("norm_odd", 1027, 1111, "rms", True, 0, False, 0.8125, quantize=False),
        # prefill of 64 prompts: norms on both sides of the block, a gate of each request's own
        _norm("norm_prefill", 19200, 2048, "rms", True, 64, False),
    ]


_HEADS = ((16, 8, 128), (16, 16, 64), (12, 12, 128), (8, 1, 128), (6, 2, 96), (9, 3, 64), (4, 4, 80), (32, 8, 128))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("attention",) * 3 + ("rotary", "norm"))
    if op == "attention":
        kind = rng.choice(("full", "causal", "causal", "cross", "tail", "tail"))
        heads, kv_heads, dim = rng.choice(_HEADS)
        batch = _log(rng, 1, 64)
        if kind in ("full", "causal"):
            # as many query-key pairs as the longest listed prompts at most
            q_hi = _log(rng, 1, int(min(8192, math.sqrt(1.3e9 / (batch * heads)))))
            k_hi = 0
        elif kind == "cross":
            q_hi, k_hi = _log(rng, 1, 128), _log(rng, 1, 1024)
        else:
            q_hi = 1 if rng.random() < 0.5 else _log(rng, 2, 64)
            k_hi = max(q_hi, _log(rng, 64, int(min(16384, 1.6e5 / batch, 1.3e9 / (batch * heads * q_hi)))))
        q_lo = 1 if q_hi == 1 else rng.choice((1, q_hi, max(1, q_hi // 3)))
        k_lo = 0 if k_hi == 0 else max(q_hi if kind == "tail" else 0, rng.choice((0, 1, k_hi // 2)))
        case = _attention("", kind, batch, q_lo, q_hi, k_lo, k_hi, heads, kv_heads, dim, rng.random() < 0.3)
    elif op == "rotary":
        heads, kv_heads, dim = rng.choice(_HEADS)
        case = _rotary("", _log(rng, 1, 20000), heads, kv_heads, dim, rng.choice((dim, dim // 2, dim // 4)),
                       rng.choice(("half", "interleaved")), rng.choice((300, 8192, 131072, 1000000)), rng.choice((1.0, 4.0, 16.0)),
                       rng.random() < 0.5)
    else:
        k = rng.choice((1024, 1536, 2048, 6144, 4096, rng.randint(64, 4096)))
        case = _norm("", _log(rng, 1, int(min(20000, 3.9e7 / k))), k, rng.choice(("rms", "layer")), rng.random() < 0.5,
                     rng.choice((0, 1, 1, 16)), rng.random() < 0.5, rng.choice((1.0, 0.8125, 0.5)), rng.random() < 0.7)
    del case["name"]
    return case


def _lengths(case):
    """Query and key lengths of a case's sequences: the first as long as the case allows, the last as short."""
    rng = random.Random(case["batch"] * 1000003 + case["q_hi"] * 1009 + case["k_hi"])
    n = case["batch"]
    lq = [case["q_hi"]] + [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(n - 1)]
    if n > 1:
        lq[-1] = case["q_lo"]
    if case["kind"] in ("full", "causal"):
        return lq, lq
    lk = [case["k_hi"]] + [rng.randint(case["k_lo"], case["k_hi"]) for _ in range(n - 1)]
    if n > 1:
        lk[-1] = case["k_lo"]
    return lq, lk


def _is_causal(case):
    return case["kind"] in ("causal", "tail")


# ----------------------------------------------------------------------------- inputs

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _heads_of(gen, tokens, counts, dim, fused):
    """One [tokens, heads, dim] tensor for each count: views of one buffer's rows, or buffers of their own."""
    rows = (_randn(gen, tokens, sum(counts) * dim) * 1.5).to(torch.bfloat16)
    parts = rows.split([c * dim for c in counts], dim=1)
    return [(p if fused else p.contiguous()).view(tokens, c, dim) for p, c in zip(parts, counts)]


def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEVICE)


def _frequencies(case):
    """Radians per position of each rotated pair, and what cosines and sines are multiplied by.  A stretched context divides the
    frequencies that turn less than once over the 4,096 positions they were made for by the factor, keeps those that turn
    32 times and more, and goes from one to the other along a ramp."""
    r, factor = case["rotary_dim"], case["factor"]
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if factor == 1.0:
        return f.to(DEVICE), 1.0
    at = lambda turns: r * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(10000.0))  # noqa: E731
    lo, hi = max(0, math.floor(at(32.0))), min(r - 1, math.ceil(at(1.0)))
    ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return (f * (1 - ramp) + f / factor * ramp).to(DEVICE), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
        if case["kind"] in ("full", "causal"):
            state["q"], state["k"], state["v"] = _heads_of(gen, sum(lq), (h, hkv, hkv), d, case["fused"])
        else:
            state["q"], = _heads_of(gen, sum(lq), (h,), d, False)
            state["k"], state["v"] = _heads_of(gen, sum(lk), (hkv, hkv), d, case["fused"])
        state["cu_q"], state["cu_k"] = _offsets(lq), _offsets(lk)
        state["most_q"], state["most_k"] = max(lq), max(lk)
    elif case["op"] == "rotary":
        t = case["tokens"]
        state["q"], state["k"] = _heads_of(gen, t, (case["heads"], case["kv_heads"]), case["dim"], case["fused"])
        state["positions"] = torch.randint(0, case["most_position"], (t,), generator=gen, device=DEVICE, dtype=torch.int32)
        state["inv_freq"], state["amplitude"] = _frequencies(case)
    else:
        m, k, rows = case["m"], case["k"], case["gate_rows"]
        bf = lambda t: t.to(torch.bfloat16)  # noqa: E731
        state["residual"] = _randn(gen, m, k)
        state["residual"][:, torch.randperm(k, generator=gen, device=DEVICE)[:max(1, k // 100)]] *= 20.0
        state["residual"], state["branch"] = bf(state["residual"]), bf(_randn(gen, m, k) * 0.7)
        state["weight"], state["post_weight"] = bf(1 + 0.1 * _randn(gen, k)), bf(1 + 0.1 * _randn(gen, k))
        state["bias"] = bf(0.1 * _randn(gen, k)) if case["norm"] == "layer" else None
        state["post_weight"] = state["post_weight"] if case["post"] else None
        vectors = max(rows, 1)
        shape = (k,) if vectors == 1 else (vectors, k)
        state["gate"] = bf(0.3 * _randn(gen, *shape)) if rows else None
        state["mod_scale"], state["mod_shift"] = (bf(0.2 * _randn(gen, *shape)) for _ in range(2)) if case["modulated"] else (None, None)
        # which request a row belongs to: requests of about the same number of rows, in order
        state["vector_rows"] = (torch.arange(m, device=DEVICE) * vectors // m).to(torch.int32) if vectors > 1 else None
    return state


# ----------------------------------------------------------------------------- one pass

@torch.no_grad()
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state)
    return _plain_attention(state) if op == "attention" else _plain_rotary(state) if op == "rotary" else _plain_norm(state)


def _run_own(state):
    from sacq_b200 import attention_packed, residual_norm_quantize_rows, rotate_heads
    case = state["case"]
    if case["op"] == "attention":
        return attention_packed(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], causal=_is_causal(case),
                                return_lse=True)
    if case["op"] == "rotary":
        return rotate_heads(state["q"], state["k"], state["positions"], state["inv_freq"], layout=case["layout"],
                            amplitude=state["amplitude"])
    return residual_norm_quantize_rows(state["branch"], state["residual"], state["weight"], state["bias"], norm=case["norm"],
                                       eps=1e-6, post_norm=case["norm"] if case["post"] else None,
                                       post_weight=state["post_weight"], gate=state["gate"],
                                       residual_scale=case["residual_scale"], mod_scale=state["mod_scale"],
                                       mod_shift=state["mod_shift"], vector_rows=state["vector_rows"],
                                       quantize=case["quantize"])


def _padded(x, cu, most):
    """[batch, heads, most, dim] of packed rows, zeros behind each sequence, and where its rows are."""
    at = torch.arange(most, device=x.device)
    lengths = (cu[1:] - cu[:-1]).long()
    real = at < lengths[:, None]
    rows = (cu[:-1, None].long() + at).clamp(max=max(x.shape[0] - 1, 0))
    return torch.where(real[..., None, None], x[rows], torch.zeros((), dtype=x.dtype, device=x.device)).permute(0, 2, 1, 3), real, lengths


def _plain_attention(state):
    case = state["case"]
    q, real_q, lq = _padded(state["q"].float(), state["cu_q"], state["most_q"])
    k, real_k, lk = _padded(state["k"].float(), state["cu_k"], state["most_k"])
    v, _, _ = _padded(state["v"].float(), state["cu_k"], state["most_k"])
    b, h, tq, d = q.shape
    hkv, tk = k.shape[1], k.shape[2]
    seen = real_k[:, None, :].expand(b, tq, tk)
    if _is_causal(case):
        i, j = torch.arange(tq, device=q.device), torch.arange(tk, device=q.device)
        seen = seen & (j <= (i + (lk - lq)[:, None])[..., None])
    s = torch.matmul(q.reshape(b, hkv, h // hkv * tq, d), k.transpose(2, 3)).view(b, hkv, h // hkv, tq, tk)
    s.mul_(1 / math.sqrt(d)).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True) if tk else s.new_full((b, hkv, h // hkv, tq, 1), -math.inf)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)            # a row that sees nothing
    p = s.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, h // hkv * tq, tk), v).view(b, hkv, h // hkv, tq, d) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).squeeze(-1).reshape(b, h, tq).permute(0, 2, 1)
    o = o.reshape(b, h, tq, d).permute(0, 2, 1, 3)
    return o[real_q].to(torch.bfloat16), lse[real_q]


def _plain_rotary(state):
    case = state["case"]
    angle = state["positions"].double()[:, None] * state["inv_freq"]           # far positions: 32 bits would lose the angle
    cos, sin = ((t * state["amplitude"]).float()[:, None, :] for t in (angle.cos(), angle.sin()))
    return tuple(_turned(state[name].float(), cos, sin, case).to(torch.bfloat16) for name in ("q", "k"))


def _turned(x, cos, sin, case):
    r = case["rotary_dim"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["layout"] == "interleaved" else (x[..., :r // 2], x[..., r // 2:r])
    y = x.clone()
    if case["layout"] == "interleaved":
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return y


def _normed(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(dim=1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * weight.float()
    return y if bias is None else y + bias.float()


def _plain_norm(state):
    case = state["case"]
    of_row = lambda t: t.float() if state["vector_rows"] is None else t.float()[state["vector_rows"].long()]  # noqa: E731
    y = state["branch"].float()
    if case["post"]:
        y = _normed(y, case["norm"], state["post_weight"], None)
    if state["gate"] is not None:
        y = y * of_row(state["gate"])
    r = state["residual"].float() * case["residual_scale"] + y
    h = _normed(r, case["norm"], state["weight"], state["bias"])
    if state["mod_scale"] is not None:
        h = h * (1 + of_row(state["mod_scale"])) + of_row(state["mod_shift"])
    if not case["quantize"]:
        return r.to(torch.bfloat16), h.to(torch.bfloat16)
    scale = h.abs().amax(dim=1, keepdim=True) / 448.0
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return r.to(torch.bfloat16), (h / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


# ----------------------------------------------------------------------------- the definitions in 64 bits

@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, state)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    return _exact_norm(case, state)


def _exact_attention(case, state):
    """out_i = sum_j softmax_j(q_i . k_j / sqrt(d)) v_j, one sequence after another."""
    d, g = case["dim"], case["heads"] // case["kv_heads"]
    lq, lk = _lengths(case)
    outs, lses, at_q, at_k = [], [], 0, 0
    for nq, nk in zip(lq, lk):
        q = state["q"][at_q:at_q + nq].double().transpose(0, 1)
        k, v = (state[n][at_k:at_k + nk].double().transpose(0, 1).repeat_interleave(g, dim=0) for n in ("k", "v"))
        logits = torch.einsum("hid,hjd->hij", q, k).mul_(d ** -0.5)
        if _is_causal(case):
            hidden = torch.ones(nq, nk, dtype=torch.bool, device=q.device).triu_(nk - nq + 1)
            logits.masked_fill_(hidden, -math.inf)
        lse = torch.logsumexp(logits, dim=2) if nk else logits.new_full((logits.shape[0], nq), -math.inf)
        w = logits.sub_(lse.masked_fill(torch.isinf(lse), 0.0)[..., None]).exp_()
        outs.append(torch.einsum("hij,hjd->ihd", w, v))
        lses.append(lse.transpose(0, 1))
        at_q, at_k = at_q + nq, at_k + nk
    return torch.cat(outs), torch.cat(lses)


def _exact_rotary(case, state):
    """A pair (a, b) as the complex number a + ib, turned by position times frequency."""
    r = case["rotary_dim"]
    turn = torch.polar(torch.full((), state["amplitude"], dtype=torch.float64, device=DEVICE).expand(case["tokens"], r // 2),
                       state["positions"].double()[:, None] * state["inv_freq"])[:, None, :]
    results = []
    for x in (state["q"].double(), state["k"].double()):
        if case["layout"] == "interleaved":
            z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:2], r // 2, 2).contiguous()) * turn
            rotated = torch.view_as_real(z).flatten(2)
        else:
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
            rotated = torch.cat([z.real, z.imag], dim=2)
        results.append(torch.cat([rotated, x[..., r:]], dim=2))
    return tuple(results)


def _exact_norm(case, state):
    def standard(x):
        centre = x.mean(1, keepdim=True) if case["norm"] == "layer" else 0.0
        return (x - centre) * ((x - centre).square().mean(1, keepdim=True) + 1e-6).rsqrt()

    each = {n: state[n].double() for n in ("gate", "mod_scale", "mod_shift") if state[n] is not None}
    if state["vector_rows"] is not None:
        each = {n: t.index_select(0, state["vector_rows"].long()) for n, t in each.items()}
    branch = state["branch"].double()
    if case["post"]:
        branch = standard(branch) * state["post_weight"].double()
    r = torch.addcmul(case["residual_scale"] * state["residual"].double(), branch, each["gate"].expand_as(branch)) if "gate" in each \
        else case["residual_scale"] * state["residual"].double() + branch
    h = standard(r) * state["weight"].double() + (0.0 if state["bias"] is None else state["bias"].double())
    if case["modulated"]:
        h = h + h * each["mod_scale"] + each["mod_shift"]
    if not case["quantize"]:
        return r, h
    largest = h.abs().max(1, keepdim=True).values
    scale = torch.where(largest > 0, largest / 448, 1.0)
    return r, (h / scale).clamp(-448, 448).to(torch.float8_e4m3fn), scale


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "attention":
        lq, lk = _lengths(case)
        h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
        pairs = 0
        for nq, nk in zip(lq, lk):
            if _is_causal(case):
                seeing = max(0, nq - max(0, nq - nk))              # queries that see a key; the last sees all nk
                pairs += seeing * nk - seeing * (seeing - 1) // 2
            else:
                pairs += nq * nk
        return {"bytes": 2.0 * d * (2 * h * sum(lq) + 2 * hkv * sum(lk)) + 4.0 * h * sum(lq) + 8.0 * (len(lq) + 1),
                "flops": 4.0 * d * h * pairs}
    if case["op"] == "rotary":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        turned = values * case["rotary_dim"] / case["dim"]
        return {"bytes": 4.0 * values + 4.0 * case["tokens"] + 4.0 * case["rotary_dim"], "flops": 3.0 * turned}
    m, k = case["m"], case["k"]
    vectors = (1 + (case["norm"] == "layer") + case["post"]) + max(case["gate_rows"], 1) * ((case["gate_rows"] > 0) + 2 * case["modulated"])
    out = 3.0 * m * k + 4.0 * m if case["quantize"] else 4.0 * m * k
    return {"bytes": 4.0 * m * k + out + 2.0 * k * vectors + (4.0 * m if case["gate_rows"] > 1 else 0), "flops": 12.0 * m * k}
