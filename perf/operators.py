"""The cases that the attention, cache-write, cache-read and cache-attention operators are measured on.

``own`` is false: ``run`` computes an operator in elementary torch operations, in 32 bits, rounded once at the end.
``own`` is true: ``run`` makes the calls that a user of evocompile_b200 makes. Both take what ``prepare`` gives.

Operators (``case["op"]``):

* ``window``   windowed attention whose first ``sinks`` keys stay visible, forward, dense [z, h, s, d]
* ``packed``   the same over packed sequences of different lengths
* ``train``    the dense form and its gradients
* ``append``   keys and values quantised into pages of a cache as they are written, and read back
* ``read``     cached sequences read back, packed
* ``attend``   attention of a few new tokens per sequence over such a cache

A cache is four tensors: codes of K and of V, uint8 [pages, kv heads, page, d * bits / 8] (4 bits: two channels a byte,
the even one in the low half), and their (scale, zero) pairs [pages, kv heads, page, 2] in the element type. A code c
stands for c * scale + zero.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
FLOOR = {"bf16": 2.0 ** -100, "f16": 2.0 ** -24}  # smallest scale of a row


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, op, dtype, z, hq, hkv, sq, sk, d, causal, window, sinks):
    return {"name": name, "op": op, "dtype": dtype, "z": z, "hq": hq, "hkv": hkv, "sq": sq, "sk": sk, "d": d,
            "causal": causal, "window": window, "sinks": sinks}


def _cache(name, op, dtype, bits, b, hq, hkv, d, page, low, high, new=1, window=0, sinks=0):
    return {"name": name, "op": op, "dtype": dtype, "bits": bits, "b": b, "hq": hq, "hkv": hkv, "d": d, "page": page,
            "low": low, "high": high, "new": new, "window": window, "sinks": sinks}


def listed():
    return [
        # a short prompt of a small model with equal heads; the smallest call
        _attention("window_short", "window", "f16", 1, 12, 12, 513, 513, 64, True, 128, 4),
        # the prompt of a 64 / 8-head block, 4096 tokens
        _attention("window_block", "window", "bf16", 1, 64, 8, 4096, 4096, 128, True, 1024, 4),
        # both directions (an encoder), more keys than queries, more sinks than one tile holds
        _attention("window_both_ways", "window", "bf16", 2, 8, 8, 1000, 1777, 128, False, 300, 131),
        # packed prompts of 31 to 2047 tokens
        dict(_attention("packed_prompts", "packed", "bf16", 6, 32, 8, 2047, 2047, 128, True, 512, 16), low=31),
        # a training step's attention, small and odd
        _attention("train_odd", "train", "f16", 2, 12, 12, 333, 333, 64, True, 100, 1),
        # a training step's attention at 4096 tokens and 32 / 8 heads
        _attention("train_4096", "train", "bf16", 1, 32, 8, 4096, 4096, 128, True, 512, 4),
        # the step of 64 sequences writes one token each
        _cache("append_step", "append", "bf16", 4, 64, 64, 8, 128, 64, 1, 1),
        # four prompts of about 4096 tokens are written
        _cache("append_prompts", "append", "f16", 8, 4, 32, 8, 128, 32, 3900, 4096),
        # sixteen cached prompts are read back for an attention over packed sequences
        _cache("read_prompts", "read", "bf16", 4, 16, 64, 8, 128, 64, 512, 8192),
        # one sequence, 131072 tokens in the cache
        _cache("attend_one_long", "attend", "bf16", 4, 1, 64, 8, 128, 64, 131072, 131072),
        # sixteen sequences of 512 to 8192 tokens answer one token each
        _cache("attend_sixteen", "attend", "bf16", 4, 16, 64, 8, 128, 64, 512, 8192),
        # five drafted tokens for each of seven sequences, 8 bits, window and sinks
        _cache("attend_drafts", "attend", "f16", 8, 7, 24, 8, 64, 16, 1, 5000, new=5, window=1000, sinks=4),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["window", "window", "packed", "train", "append", "read", "attend", "attend", "attend"])
    dtype, d = rng.choice(["bf16", "f16"]), rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op in ("window", "packed", "train"):
        group = rng.choice([1, 2, 4, 8])
        sk = sq = _log(rng, 64, 2048 if op != "window" else 4096)
        causal = rng.random() < 0.8
        if op != "packed" and rng.random() < 0.2:
            sk = _log(rng, 64, 2048)
        z = rng.randint(2, 9) if op == "packed" else rng.choice([1, 1, 2, 3])
        while z * hkv * group > 48 and group > 1:
            group //= 2
        case = _attention("", op, dtype, z, hkv * group, hkv, sq, sk, d, causal, _log(rng, 16, 1500), _log(rng, 1, 200))
        if op == "packed":
            case["low"] = rng.randint(1, sq)
    else:
        b, new, group = _log(rng, 1, 32), 1, rng.choice([1, 2, 3, 4, 7, 8])
        high = _log(rng, 1, 16384 if b > 4 else 65536)
        if op == "append":
            high = _log(rng, 1, max(1, 16384 // b))
        if op == "read":
            high = _log(rng, 1, max(1, 60000 // b))
        window, sinks = (_log(rng, 16, 4096), _log(rng, 1, 100)) if rng.random() < 0.4 else (0, 0)
        if op == "attend":
            new = rng.choice([1, 1, 1, 2, 5, 16])
            while b * high * hkv * group * new > 64 * 131072 and new > 1:
                new //= 2
            while b * high * hkv * max(group * new, 8) > 64 * 131072 and high > 1:
                high //= 2
        else:
            window = sinks = 0
        case = _cache("", op, dtype, rng.choice([4, 8]), b, hkv * group, hkv, d, rng.choice([16, 32, 64, 128]),
                      rng.randint(1, high), high, new, window, sinks)
    del case["name"]
    return case


def _lengths(case, seed):
    """Tokens of each sequence, between ``low`` and ``high`` (both met): a case's own, their order by the seed."""
    low, high, n = case["low"], case["high"] if "high" in case else case["sq"], case["b"] if "b" in case else case["z"]
    got = np.random.RandomState(low * 31 + high * 7 + n).randint(low, high + 1, n)
    got[0] = high
    if n > 1:
        got[1] = low
    return np.random.RandomState(seed % (1 << 31)).permutation(got)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def keys(*lead):  # keys have channels of their own mean, as rotated keys of real models do
        return (normal(*lead, hkv, d) + 1.5 * normal(hkv, d)).to(dtype)

    state = {"case": case, "scale": d ** -0.5}
    if case["op"] == "packed":
        lens = _lengths(case, seed)
        cu = np.concatenate([[0], np.cumsum(lens)])
        t = int(cu[-1])
        state.update(q=normal(t, hq, d).to(dtype), k=keys(t), v=normal(t, hkv, d).to(dtype),
                     cu=torch.tensor(cu, dtype=torch.int32, device=dev), longest=int(lens.max()))
        return state
    if case["op"] in ("window", "train"):
        # storage [z, s, h, d], as a projection leaves it, seen as [z, h, s, d]
        z, sq, sk = case["z"], case["sq"], case["sk"]
        state.update(q=normal(z, sq, hq, d).to(dtype).transpose(1, 2), k=keys(z, sk).transpose(1, 2),
                     v=normal(z, sk, hkv, d).to(dtype).transpose(1, 2))
        if case["op"] == "train":
            state["dout"] = normal(z, sq, hq, d).to(dtype).transpose(1, 2)
            for n in "qkv":
                state[n].requires_grad_(True)
        return state
    # a cache whose pages belong to the sequences in no order, with a few pages that belong to none
    lens, page, b = _lengths(case, seed), case["page"], case["b"]
    if case["op"] == "attend":
        lens = np.maximum(lens, 1)
    width = -(-int(lens.max()) // page)
    need = -(-lens // page)
    pages = int(need.sum()) + 3
    free = np.random.RandomState((seed + 1) % (1 << 31)).permutation(pages)
    table, at = np.zeros((b, width), np.int32), 0
    for i in range(b):
        table[i, :need[i]] = free[at:at + need[i]]
        at += need[i]
    total = int(lens.sum())
    cu = np.concatenate([[0], np.cumsum(lens)])
    state.update(table=torch.tensor(table, device=dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                 cu=torch.tensor(cu, dtype=torch.int32, device=dev), total=total, longest=int(lens.max()))
    if case["op"] == "append":
        row = np.repeat(np.arange(b), lens)
        pos = np.arange(total) - cu[row]
        slots = table[row, pos // page].astype(np.int64) * page + pos % page
        width_bytes = d * case["bits"] // 8
        state.update(k=keys(total), v=normal(total, hkv, d).to(dtype), slots=torch.tensor(slots, device=dev),
                     cache=(torch.zeros(pages, hkv, page, width_bytes, dtype=torch.uint8, device=dev),
                            torch.zeros(pages, hkv, page, width_bytes, dtype=torch.uint8, device=dev),
                            torch.zeros(pages, hkv, page, 2, dtype=dtype, device=dev),
                            torch.zeros(pages, hkv, page, 2, dtype=dtype, device=dev)))
        return state
    ck, pk = _quantise(keys(pages, page).transpose(1, 2).contiguous(), case["bits"], case["dtype"])
    cv, pv = _quantise(normal(pages, hkv, page, d).to(dtype), case["bits"], case["dtype"])
    state["cache"] = (_pack(ck, case["bits"]), _pack(cv, case["bits"]), pk, pv)
    if case["op"] == "attend":
        new = case["new"]
        state.update(q=normal(b * new, hq, d).to(dtype),
                     cu_q=torch.arange(0, b * new + 1, new, dtype=torch.int32, device=dev))
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x, bits, kind):
    """Codes (uint8) and (scale, zero) pairs of rows x [..., d], in 32 bits."""
    f = x.float()
    low, high = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    scale = (high - low) / torch.full_like(high, 2 ** bits - 1)  # by a tensor: by a number it would be a product
    near = scale.to(x.dtype)
    up = (near.view(torch.int16) + 1).view(x.dtype)  # the next one above, for what was rounded down
    scale = torch.where(near.float() < scale, up, near).float().clamp_min(FLOOR[kind])
    codes = torch.round((f - low) / scale).clamp(0, 2 ** bits - 1).to(torch.uint8)
    return codes, torch.cat([scale, low], -1).to(x.dtype)


def _pack(codes, bits):
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(codes, bits):
    return codes if bits == 8 else torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, pairs, bits):
    """What codes [..., d * bits / 8] with pairs [..., 2] stand for, in 32 bits."""
    pairs = pairs.float()
    return _unpack(codes, bits).float() * pairs[..., :1] + pairs[..., 1:]


def _softmax(s, keep):
    """(P, lse) over the last axis of logits s where keep; a row with nothing kept gives zeros and -inf."""
    s = s.masked_fill(~keep, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    return p, (m + torch.log(total)).squeeze(-1)


def _visible(i, j, case):
    keep = torch.ones_like(i + j, dtype=torch.bool)
    if case["window"]:
        keep = ((i - j).abs() <= case["window"]) | (j < case["sinks"])
    return keep & (j <= i) if case.get("causal", True) else keep


def _dense(q, k, v, keep, scale):
    """Attention of 32-bit q [z, hq, sq, d] over k, v [z, hkv, sk, d]: (out, lse [z * hq, sq])."""
    z, hq, sq, d = q.shape
    hkv, sk = k.shape[1:3]
    s = torch.matmul(q.reshape(z, hkv, -1, d), k.transpose(-1, -2)).view(z, hkv, hq // hkv, sq, sk) * scale
    p, lse = _softmax(s, keep)
    out = torch.matmul(p.view(z, hkv, -1, sk), v).view(z, hq, sq, d)
    return out, lse.reshape(z * hq, sq)


def _plain(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    op, hq, hkv, d = case["op"], case["hq"], case["hkv"], case["d"]
    if op == "packed":
        q, k, v = (state[n].float().transpose(0, 1)[None] for n in "qkv")
        at = torch.arange(q.shape[2], device=q.device, dtype=torch.int32)
        seq = torch.searchsorted(state["cu"][1:], at, right=True)
        pos = at - state["cu"][seq]
        keep = (seq[:, None] == seq[None, :]) & _visible(pos[:, None], pos[None, :], case)
        out, lse = _dense(q, k, v, keep, state["scale"])
        return out[0].transpose(0, 1).to(dtype), lse
    if op in ("window", "train"):
        q, k, v = state["q"], state["k"], state["v"]
        i, j = (torch.arange(n, device=q.device) for n in (q.shape[2], k.shape[2]))
        keep = _visible(i[:, None], j[None, :], case)
        if op == "window":
            out, lse = _dense(q.float(), k.float(), v.float(), keep, state["scale"])
            return out.to(dtype), lse
        leaves = [t.detach().float().requires_grad_(True) for t in (q, k, v)]
        out, _ = _dense(*leaves, keep, state["scale"])
        grads = torch.autograd.grad(out, leaves, state["dout"].float())
        return [t.detach().to(dtype) for t in (out, *grads)]
    bits, page = case["bits"], case["page"]
    if op == "append":
        back, at, row = [], state["slots"] // page, state["slots"] % page
        for x, codes_to, pairs_to in ((state["k"], 0, 2), (state["v"], 1, 3)):
            codes, pairs = _quantise(x, bits, case["dtype"])
            codes_to, pairs_to = state["cache"][codes_to], state["cache"][pairs_to]
            codes_to[at, :, row] = _pack(codes, bits)
            pairs_to[at, :, row] = pairs
            back.append(_values(codes_to[at, :, row], pairs_to[at, :, row], bits).to(dtype))
        return back
    ck, cv, pk, pv = state["cache"]
    if op == "read":
        at = torch.arange(state["total"], device=ck.device, dtype=torch.int32)
        seq = torch.searchsorted(state["cu"][1:], at, right=True)
        pos = (at - state["cu"][seq]).long()
        where, row = state["table"][seq, pos // page].long(), pos % page
        return [_values(c[where, :, row], p[where, :, row], bits).to(dtype) for c, p in ((ck, pk), (cv, pv))]
    # attend: the pages of each sequence in order, then one batched attention over the longest
    b, new, table = case["b"], case["new"], state["table"].long()
    k, v = (_values(c[table], p[table], bits).transpose(1, 2).reshape(b, hkv, -1, d) for c, p in ((ck, pk), (cv, pv)))
    q = state["q"].float().view(b, new, hq, d).transpose(1, 2)
    i = (state["lens"][:, None] - new + torch.arange(new, device=q.device))[:, :, None]
    j = torch.arange(k.shape[2], device=q.device)[None, None, :]
    keep = (_visible(i, j, case) & (j < state["lens"][:, None, None]))[:, None, None]
    out, lse = _dense(q, k, v, keep, state["scale"])
    return out.transpose(1, 2).reshape(b * new, hq, d).to(dtype), lse.view(b, hq, new).transpose(0, 1).reshape(hq, -1)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if not own:
        return _plain(state)
    from evocompile_b200 import ops
    from evocompile_b200.kernels import fused_sdpa

    case = state["case"]
    op, window, sinks = case["op"], case["window"], case["sinks"]
    if op == "window":
        return ops.fmha_fwd(state["q"], state["k"], state["v"], None, state["scale"], int(case["causal"]), window,
                            sinks=sinks)
    if op == "packed":
        return ops.fmha_varlen_fwd(state["q"], state["k"], state["v"], state["cu"], state["cu"], state["longest"],
                                   state["longest"], state["scale"], int(case["causal"]), window, sinks=sinks)
    if op == "train":
        leaves = state["q"], state["k"], state["v"]
        out = fused_sdpa.fused_attention(*leaves, None, state["scale"], int(case["causal"]), window, sinks=sinks)
        return [out.detach(), *torch.autograd.grad(out, leaves, state["dout"])]
    if op == "append":
        ops.kv_cache_write(state["k"], state["v"], state["cache"], state["slots"])
        return ops.kv_cache_read(state["cache"], state["table"], state["cu"], state["total"], case["d"])
    if op == "read":
        return ops.kv_cache_read(state["cache"], state["table"], state["cu"], state["total"], case["d"])
    return ops.fmha_cache_fwd(state["q"], state["cache"], state["table"], state["lens"], state["cu_q"], case["new"],
                              state["longest"], state["scale"], 1, window, sinks=sinks)


# ------------------------------------------------------------------------------------------------ what a pass needs
def _pairs(case, length_q, length_k, offset=0):
    """Visible (query, key) pairs of one sequence and head; query i stands at offset + i."""
    i = np.arange(length_q, dtype=np.int64) + offset
    last = np.minimum(length_k, i + 1) if case.get("causal", True) else np.full_like(i, length_k)
    last = np.maximum(last, 0)
    if not case["window"]:
        return int(last.sum())
    low = np.clip(i - case["window"], 0, last)
    high = np.clip(i + case["window"] + 1, low, last)
    return int((high - low + np.minimum(np.minimum(case["sinks"], low), last)).sum() +
               np.maximum(0, np.minimum(case["sinks"], last) - high).sum())


def work(case):
    op, hq, hkv, d = case["op"], case["hq"], case["hkv"], case["d"]
    if op in ("window", "train"):
        z, sq, sk = case["z"], case["sq"], case["sk"]
        pairs = z * hq * _pairs(case, sq, sk)
        q, kv = 2 * z * hq * sq * d, 2 * z * hkv * sk * d
        if op == "window":
            return {"bytes": 2 * q + 2 * kv + 4 * z * hq * sq, "flops": 4 * d * pairs}
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * d * pairs}
    lens = _lengths(case, 0)
    tokens = int(lens.sum())
    if op == "packed":
        return {"bytes": 2 * tokens * d * (2 * hq + 2 * hkv) + 4 * hq * tokens,
                "flops": 4 * d * hq * sum(_pairs(case, int(n), int(n)) for n in lens)}
    row = d * case["bits"] // 8 + 4
    if op == "append":
        return {"bytes": 2 * tokens * hkv * (2 * d + 2 * row + 2 * d) + 8 * tokens, "flops": 8 * tokens * hkv * d}
    if op == "read":
        return {"bytes": 2 * tokens * hkv * (row + 2 * d), "flops": 4 * tokens * hkv * d}
    lens, new = np.maximum(lens, 1), case["new"]
    seen = sum(int(n) if not case["window"] else min(int(n), case["window"] + new + case["sinks"]) for n in lens)
    return {"bytes": 2 * seen * hkv * row + 4 * case["b"] * new * hq * d + 4 * case["b"] * new * hq,
            "flops": 4 * d * hq * sum(_pairs(case, new, int(n), int(n) - new) for n in lens)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows(case, codes, pairs):
    """Dequantised rows in 64 bits, channel by channel from the definition."""
    pairs = pairs.double()
    if case["bits"] == 8:
        c = codes.double()
    else:
        c = torch.empty(*codes.shape[:-1], case["d"], dtype=torch.float64, device=codes.device)
        c[..., 0::2] = torch.remainder(codes, 16).double()
        c[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    return c * pairs[..., 0:1] + pairs[..., 1:2]


def _exact_head(q, k, v, i, case, scale, dout=None):
    """One head in 64 bits: out and lse, and with dout the gradients by their formulas."""
    j = torch.arange(k.shape[0], device=q.device)
    hidden = torch.zeros(q.shape[0], k.shape[0], dtype=torch.bool, device=q.device)
    if case["window"]:
        hidden = (torch.abs(i[:, None] - j[None, :]) > case["window"]) & (j[None, :] >= case["sinks"])
    if case.get("causal", True):
        hidden = hidden | (j[None, :] > i[:, None])
    s = (q @ k.T * scale).masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, 1)
    p = torch.where(hidden, 0.0, torch.exp(s - lse[:, None]))
    out = p @ v
    if dout is None:
        return out, lse
    ds = p * (dout @ v.T - (out * dout).sum(1, keepdim=True)) * scale
    return out, ds @ k, ds.T @ q, p.T @ dout


def exact(case, seed):
    state = prepare(case, seed)
    op, hq, hkv, d, scale = case["op"], case["hq"], case["hkv"], case["d"], state["scale"]
    group = hq // hkv
    if op in ("window", "train"):
        q, k, v = (state[n].detach().double() for n in "qkv")
        z, sq = q.shape[0], q.shape[2]
        i = torch.arange(sq, device=q.device)
        if op == "window":
            got = [_exact_head(q[b, h], k[b, h // group], v[b, h // group], i, case, scale)
                   for b in range(z) for h in range(hq)]
            return torch.stack([x[0] for x in got]).view(z, hq, sq, d), torch.stack([x[1] for x in got])
        out, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
        for b in range(z):
            for h in range(hq):
                o, a, c, e = _exact_head(q[b, h], k[b, h // group], v[b, h // group], i, case, scale,
                                         state["dout"][b, h].double())
                out[b, h], dq[b, h] = o, a
                dk[b, h // group] += c
                dv[b, h // group] += e
        return [out, dq, dk, dv]
    if op == "packed":
        q, k, v = (state[n].double() for n in "qkv")
        out = torch.empty_like(q)
        lse = torch.empty(hq, q.shape[0], dtype=torch.float64, device=q.device)
        cu = state["cu"].tolist()
        for a, e in zip(cu[:-1], cu[1:]):
            i = torch.arange(e - a, device=q.device)
            for h in range(hq):
                out[a:e, h], lse[h, a:e] = _exact_head(q[a:e, h], k[a:e, h // group], v[a:e, h // group], i, case, scale)
        return out, lse
    if op == "append":
        back = []
        for x in (state["k"].double(), state["v"].double()):
            low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
            wide = (high - low) / (2 ** case["bits"] - 1)
            # the smallest value of the element type that is not below: 8 (11) significant bits
            step = torch.exp2(torch.floor(torch.log2(wide.clamp_min(2.0 ** -200))) - (7 if case["dtype"] == "bf16" else 10))
            if case["dtype"] == "f16":
                step = step.clamp_min(2.0 ** -24)
            scale_row = (torch.ceil(wide / step) * step).clamp_min(FLOOR[case["dtype"]])
            codes = torch.round((x - low) / scale_row).clamp(0, 2 ** case["bits"] - 1)
            back.append(codes * scale_row + low)
        return back
    cu = state["cu"].tolist()
    seqs = []
    for b in range(case["b"]):
        n, page = cu[b + 1] - cu[b], case["page"]
        used = state["table"][b, :-(-n // page)].long()
        ck, cv, pk, pv = (t[used].transpose(1, 2).flatten(0, 1)[:n] for t in state["cache"])
        seqs.append((_exact_rows(case, ck, pk), _exact_rows(case, cv, pv)))
    if op == "read":
        return [torch.cat([s[n] for s in seqs]) for n in (0, 1)]
    new = case["new"]
    q = state["q"].double()
    out = torch.zeros_like(q)
    lse = torch.empty(hq, q.shape[0], dtype=torch.float64, device=q.device)
    for b, (k, v) in enumerate(seqs):
        rows = slice(b * new, (b + 1) * new)
        i = k.shape[0] - new + torch.arange(new, device=q.device)
        for h in range(hq):
            o, l = _exact_head(q[rows, h], k[:, h // group], v[:, h // group], i, case, scale)
            out[rows, h], lse[h, rows] = torch.where(l[:, None] == -math.inf, 0.0, o), l
    return out, lse
