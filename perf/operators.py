"""The attention operators behind the projection front, as a serving program calls them.

Prompts are attended over as they come from ``fused_qkv_rope`` (packed, causal, grouped
heads); their keys and values go into a paged cache of 4-bit codes; decode steps attend
over that cache, and may sum up each key's attention weight; and a sequence that outgrows
its budget drops the keys with the least weight.  The shapes are the Qwen3 ones the tests
and the benchmark use.  ``run`` computes every operator in elementary torch operations,
or calls the framework's where ``own`` is true.

The 4-bit cache.  A page holds 16 tokens; of a page, one key / value head has a record of
18 D bytes (D = 64 or 128), held as 9 D elements of the model's type:

  K codes  8 D bytes  [quarter 4][token 16][group D/64][2][8 codes]: dimension
           64 group + 16 quarter + 8 half + j, code j = 2 i at nibble i of its four
           bytes and j = 2 i + 1 at nibble i + 4
  V codes  8 D bytes  [token / 4][m 16][token % 4][group D/64][4 codes]: dimension
           64 group + 4 m + b at nibble b of its two bytes
  K, V     D bytes each  [token 16][group D/64][scale, least], of the model's type

A group of 64 dimensions of one token's head has least = its smallest value and scale =
(largest - smallest) / 15, rounded to float32 and then to the model's type; a code is
(x - least) / scale to the nearest whole number, ties to the even one, within 0 .. 15
(0 where the scale is 0), and stands for scale * code + least.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# (query heads, key / value heads): Qwen3-0.6B / 1.7B, 4B / 8B, 30B-A3B, 14B, 235B-A22B
HEADS = [(16, 8), (32, 8), (32, 4), (40, 8), (64, 4)]
MOST_FLOPS = 5.4e11   # of a drawn prompt: the largest listed case's
MOST_KEYS = 2.2e6     # keys times key / value heads of a drawn decode step


def _mqk():
    pkg = os.path.join(os.getcwd(), "mini-qwen-llm_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mqk
    return mqk


# --- the cases ---------------------------------------------------------------------------


def _prompt(T, seqs, heads, kind="bf16", D=128, prefix=0):
    return {"op": "prompt", "T": T, "seqs": seqs, "hq": heads[0], "hkv": heads[1], "kind": kind, "D": D,
            "prefix": prefix}


def _store(T, seqs, hkv, kind="bf16", D=128, context=0):
    return {"op": "store", "T": T, "seqs": seqs, "hkv": hkv, "kind": kind, "D": D, "context": context}


def _decode(seqs, context, heads, kind="bf16", D=128, tokens=1, weights=False):
    return {"op": "decode", "seqs": seqs, "context": context, "hq": heads[0], "hkv": heads[1], "kind": kind, "D": D,
            "tokens": tokens, "weights": weights}


def _evict(seqs, context, hkv, budget, recent, kind="bf16", D=128):
    return {"op": "evict", "seqs": seqs, "context": context, "hkv": hkv, "kind": kind, "D": D, "budget": budget,
            "recent": recent}


def listed():
    return [
        # the reference's CPU-runnable layer in its own type: one short prompt, latency
        {"name": "prompt_f32_0.6b_s128", **_prompt(128, 1, (16, 8), "f32")},
        # the default configuration (head_dim 64) loaded in fp16, a batch of prompts
        {"name": "prompt_f16_hd64_4x512", **_prompt(2048, 4, (16, 8), "f16", 64)},
        # a ragged continuous batch of prompts at Qwen3-8B size
        {"name": "prompt_8b_ragged_t8214", **_prompt(8214, 16, (32, 8))},
        # the next 1024 tokens of a long prompt, over the 7000 that are there already
        {"name": "prompt_8b_1024_after_7000", **_prompt(1024, 1, (32, 8), prefix=7000)},
        # one long prompt at 30B-A3B size: the largest product
        {"name": "prompt_30b_s8192", **_prompt(8192, 1, (32, 4))},
        # the keys and values of that ragged batch into the cache, and back
        {"name": "store_8b_ragged_t8214", **_store(8214, 16, 8)},
        # one decode step's tokens into the cache: latency
        {"name": "store_8b_step_b64", **_store(64, 64, 8, context=4096)},
        # one token of one sequence, the smallest model
        {"name": "decode_0.6b_b1_c300", **_decode(1, 300, (16, 8))},
        # a decode step of 64 ragged sequences at Qwen3-8B size: the cache's bytes
        {"name": "decode_8b_b64_c8192", **_decode(64, 8192, (32, 8))},
        # a few long sequences that keep count of their keys' weights
        {"name": "decode_30b_b4_c32768_weights", **_decode(4, 32768, (32, 4), weights=True)},
        # one long sequence back to its budget
        {"name": "evict_8b_b1_c4096", **_evict(1, 4096, 8, 2048, 64)},
        # a batch of sequences back to their budget
        {"name": "evict_8b_b32_c6000", **_evict(32, 6000, 8, 2048, 128)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "store", "decode", "decode", "evict"])
    kind = rng.choice(["bf16", "bf16", "bf16", "f16"])
    heads = rng.choice(HEADS)
    D = rng.choice([128, 128, 128, 64])
    if op == "prompt":
        kind = rng.choice(["bf16", "bf16", "bf16", "bf16", "f16", "f16", "f32"])
        D = rng.choice([128, 128, 128, 128, 64, 64, 80, 96, 256])
        seqs = rng.choice([1, 1, 2, 3, 4, 7, 16])
        prefix = rng.choice([0, 0, 0, _log_int(rng, 16, 4000)])
        most = 1024 if kind == "f32" else 8192
        while True:
            case = _prompt(_log_int(rng, 40, most), seqs, heads, kind, D, prefix)
            if case["T"] >= 8 * seqs and _plain_pairs(case) * 4.0 * D * heads[0] <= 2 * MOST_FLOPS:
                return case
    if op == "store":
        if rng.random() < 0.5:
            return _store(_log_int(rng, 40, 8192), rng.choice([1, 2, 5, 16]), heads[1], kind, D)
        seqs = _log_int(rng, 1, 128)
        return _store(seqs, seqs, heads[1], kind, D, context=_log_int(rng, 16, 8192))
    if op == "decode":
        seqs = _log_int(rng, 1, 128)
        context = _log_int(rng, 20, max(21, min(40000, int(MOST_KEYS / seqs / heads[1]))))
        return _decode(seqs, context, heads, kind, D, rng.choice([1, 1, 1, 1, 2, 5]), rng.random() < 0.3)
    seqs = _log_int(rng, 1, 32)
    context = _log_int(rng, 64, 8192)
    budget = max(16, int(context * rng.uniform(0.2, 0.9)))
    return _evict(seqs, context, heads[1], budget, rng.randint(0, budget // 4), kind, D)


def _shares(total, n, key):
    """``total`` over ``n`` sequences, each within a factor of about three of the others."""
    rng = random.Random("%s %d %d" % (key, total, n))
    w = [rng.uniform(0.5, 1.5) for _ in range(n)]
    at = [round(total * sum(w[:i]) / sum(w)) for i in range(n + 1)]
    return [b - a for a, b in zip(at, at[1:])]


def _lens(case):
    """Tokens of each sequence: (new ones, all of them)."""
    op, n = case["op"], case["seqs"]
    if op == "prompt":
        equal = case["T"] % n == 0 and case["T"] // n == 512
        new = [512] * n if equal else _shares(case["T"], n, "prompt")
        return new, [x + case["prefix"] for x in new]
    if op == "store":
        if not case["context"]:
            new = _shares(case["T"], n, "store")
            return new, new
        rng = random.Random("store %d %d" % (n, case["context"]))
        return [1] * n, [rng.randint(1, case["context"]) for _ in range(n)]
    rng = random.Random("%s %d %d" % (op, n, case["context"]))
    least = max(case.get("tokens", 1), case["context"] // 4)
    total = [max(least, case["context"])] + [rng.randint(least, max(least, case["context"])) for _ in range(n - 1)]
    return [case.get("tokens", 1)] * n, total


def _pairs(case):
    new, total = _lens(case)
    return sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))


def _plain_pairs(case):
    """Pairs of the padded plain form."""
    new, total = _lens(case)
    return len(new) * max(new) * max(total)


def work(case):
    new, total = _lens(case)
    size = 4 if case["kind"] == "f32" else 2
    D, hkv = case["D"], case["hkv"]
    record = hkv * 18 * D // PAGE  # bytes of one token in the cache
    if case["op"] == "prompt":
        hq = case["hq"]
        return {"bytes": (2 * hq * sum(new) + 2 * hkv * sum(total)) * D * size, "flops": 4 * D * hq * _pairs(case)}
    if case["op"] == "store":
        return {"bytes": sum(new) * (4 * hkv * D * size + record), "flops": sum(new) * hkv * D * 12}
    if case["op"] == "decode":
        hq, s = case["hq"], case["tokens"]
        weights = 8 * hkv * sum(total) if case["weights"] else 0
        return {"bytes": sum(total) * record + 2 * len(new) * s * hq * D * size + weights,
                "flops": 4 * D * hq * _pairs(case)}
    kept = sum(min(t, case["budget"]) for t in total if t > case["budget"])
    back = sum(min(t, case["budget"]) for t in total)
    return {"bytes": 4 * hkv * sum(total) + kept * (2 * record + 4 * hkv) + back * 2 * hkv * D * size,
            "flops": 4 * hkv * sum(total)}


# --- inputs ------------------------------------------------------------------------------


def _offsets(lens, dev):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["kind"]]
    D, hkv, hq = case["D"], case["hkv"], case.get("hq", 0)
    new, total = _lens(case)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dt)

    st = {"case": case, "scale": D ** -0.5, "new": new, "total": total, "cu": _offsets(new, dev)}
    if case["op"] == "prompt":
        # q as the norm leaves it with a gain of 2: some keys stand out, as they do in earnest
        st.update(q=normal(sum(new), hq, D, std=2.0), k=normal(sum(total), hkv, D), v=normal(sum(total), hkv, D))
        st["cu_k"] = _offsets(total, dev) if case["prefix"] else None
        return st
    # every sequence has pages of its own, in no order; a few pages belong to nobody
    pages = [-(-t // PAGE) for t in total]
    cols, count = max(pages), sum(pages) + 3
    ids = torch.randperm(count, generator=g, device=dev)[:sum(pages)].to(torch.int32)
    rows = torch.tensor([i for i, n in enumerate(pages) for _ in range(n)], device=dev)
    at = torch.tensor([j for n in pages for j in range(n)], device=dev)
    table = torch.zeros(len(pages), cols, dtype=torch.int32, device=dev)
    table[rows, at] = ids
    st.update(table=table, lens=torch.tensor(total, dtype=torch.int32, device=dev), rows=rows, at=at)
    st["weights"] = None
    if case["op"] == "store":
        st.update(k=normal(sum(new), hkv, D), v=normal(sum(new), hkv, D))
        st["cache"] = torch.zeros(count, hkv, 9 * D, dtype=dt, device=dev)
        if case["context"]:
            st["weights"] = torch.rand(count, hkv, PAGE, generator=g, device=dev)
        return st
    gain = (1 + 0.3 * torch.rand(D, generator=g, device=dev)).to(dt)  # channels differ in size
    k = normal(count * PAGE, hkv, D) * gain
    codes_k = _quantise(k, torch.float32)
    del k
    codes_v = _quantise(normal(count * PAGE, hkv, D), torch.float32)
    st["cache"] = _pack(*codes_k, *codes_v)
    if case["op"] == "decode":
        st["q"] = normal(len(new), case["tokens"], hq, D, std=2.0)
        if case["weights"]:
            st["weights"] = torch.rand(count, hkv, PAGE, generator=g, device=dev)
        return st
    # weights as a decode run leaves them: a few keys hold most of it
    st["weights"] = torch.rand(count, hkv, PAGE, generator=g, device=dev).pow(6) * 8
    kept = [min(t, case["budget"]) for t in total]
    st.update(kept=sum(kept), cu_kept=_offsets(kept, dev))
    return st


# --- the operators -----------------------------------------------------------------------


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        mqk = _mqk()
        if op == "prompt":
            return mqk.attn_prefill(st["q"], st["k"], st["v"], st["cu"], cu_seqlens_k=st["cu_k"])
        if op == "store":
            mqk.kv4_write(st["k"], st["v"], st["cache"], st["table"], st["lens"], cu_seqlens=st["cu"],
                          scores=st["weights"])
            k, v = mqk.kv4_read(st["cache"], st["table"], st["lens"], st["k"].shape[0], cu_seqlens=st["cu"])
            return {"k": k, "v": v, "weights": st["weights"]}
        if op == "decode":
            out = mqk.kv4_attn(st["q"], st["cache"], st["table"], st["lens"], scores=st["weights"])
            return {"out": out, "weights": st["weights"]}
        lens, kept = mqk.kv4_evict(st["cache"], st["weights"], st["table"], st["lens"], case["budget"],
                                   recent=case["recent"])
        k, v = mqk.kv4_read(st["cache"], st["table"], lens, st["kept"], cu_seqlens=st["cu_kept"])
        return {"lens": lens, "kept": kept, "k": k, "v": v, "weights": st["weights"]}
    return {"prompt": _plain_prompt, "store": _plain_store, "decode": _plain_decode, "evict": _plain_evict}[op](st)


def _token_rows(cu, n):
    """Sequence and place in it of every packed token."""
    t = torch.arange(n, device=cu.device)
    s = torch.searchsorted(cu[1:].long(), t, right=True)
    return s, t - cu.long()[s]


def _attend(q, k, v, limit, scale):
    """q [B, S, Hq, D], k / v [B, L, Hkv, D] in float32, limit [B, S]: the keys each query sees.
    The weights [B, Hq, S, L] and the output [B, S, Hq, D]; a query that sees no key gets 0."""
    G = q.shape[2] // k.shape[2]
    k, v = (x.permute(0, 2, 1, 3).repeat_interleave(G, 1) for x in (k, v))
    s = torch.matmul(q.permute(0, 2, 1, 3), k.transpose(2, 3)) * scale
    seen = torch.arange(k.shape[2], device=q.device) < limit[:, None, :, None]
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return p, torch.matmul(p, v).permute(0, 2, 1, 3)


def _plain_prompt(st):
    q, cu = st["q"], st["cu"]
    cu_k = cu if st["cu_k"] is None else st["cu_k"]
    B, S, L = len(st["new"]), max(st["new"]), max(st["total"])
    sq, pq = _token_rows(cu, q.shape[0])
    sk, pk = _token_rows(cu_k, st["k"].shape[0])
    qp = torch.zeros(B, S, *q.shape[1:], device=q.device)
    qp[sq, pq] = q.float()
    kp, vp = (torch.zeros(B, L, *st["k"].shape[1:], device=q.device) for _ in range(2))
    kp[sk, pk], vp[sk, pk] = st["k"].float(), st["v"].float()
    n, m = cu.diff().long(), cu_k.diff().long()
    limit = (m - n)[:, None] + 1 + torch.arange(S, device=q.device)
    return _attend(qp, kp, vp, limit, st["scale"])[1][sq, pq].to(q.dtype)


def _quantise(x, bits=torch.float64):
    """x [N, H, D]: codes uint8 [N, H, D], and scale and least [N, H, D / 64] of x's type.
    (64 bits: a value next to the border between two codes, and the border itself.)"""
    g = x.to(bits).unflatten(-1, (-1, 64))
    lo, hi = g.aminmax(dim=-1)
    scale = ((hi - lo) / 15).float().to(x.dtype)
    s = scale.to(bits)[..., None]
    codes = torch.where(s > 0, ((g - lo[..., None]) / s).round().clamp(0, 15), 0)
    return codes.to(torch.uint8).flatten(-2), scale, lo.to(x.dtype)


def _pack(kc, ks, kl, vc, vs, vl):
    """Whole pages of codes [16 P, H, D] and their scales and least values as records [P, H, 9 D]."""
    n, H, D = kc.shape
    P, G = n // PAGE, D // 64
    # K: token, group, quarter, half, i, parity -> quarter, token, group, half, parity, i
    k = kc.view(P, PAGE, H, G, 4, 2, 4, 2).permute(0, 2, 4, 1, 3, 5, 7, 6).reshape(P, H, -1, 2)
    # V: token / 4, token % 4, group, m, b -> token / 4, m, token % 4, group, b
    v = vc.view(P, 4, 4, H, G, 16, 4).permute(0, 3, 1, 5, 2, 4, 6).reshape(P, H, -1, 2)
    codes = [(c[..., 0] | c[..., 1] << 4).contiguous().view(ks.dtype) for c in (k, v)]
    meta = [torch.stack(x, -1).view(P, PAGE, H, G, 2).transpose(1, 2).reshape(P, H, -1) for x in ((ks, kl), (vs, vl))]
    return torch.cat(codes + meta, -1)


def _codes(records):
    """Records [..., H, 9 D]: codes of K and V [..., 16, H, D] (uint8), their scales and least
    values [..., 16, H, D / 64]."""
    lead, D = records.shape[:-2], records.shape[-1] // 9
    G, r = D // 64, records.contiguous().flatten(0, -3)
    P, H = r.shape[:2]
    b = r[..., :8 * D].contiguous().view(torch.uint8).view(P, H, 2, 8 * D)
    b = torch.stack((b & 15, b >> 4), -1)
    k = b[:, :, 0].reshape(P, H, 4, PAGE, G, 2, 2, 4).permute(0, 3, 1, 4, 2, 5, 7, 6)
    v = b[:, :, 1].reshape(P, H, 4, 16, 4, G, 4).permute(0, 2, 4, 1, 5, 3, 6)
    m = r[..., 8 * D:].view(P, H, 2, PAGE, G, 2).permute(2, 5, 0, 3, 1, 4)
    k, v = (x.reshape(*lead, PAGE, H, D) for x in (k, v))
    (ks, kl), (vs, vl) = (tuple(x.reshape(*lead, PAGE, H, G) for x in pair) for pair in m)
    return k, ks, kl, v, vs, vl


def _values(codes, scale, least):
    g = codes.float().unflatten(-1, (-1, 64))
    return (g * scale.float()[..., None] + least.float()[..., None]).flatten(-2)


def _plain_store(st):
    k, cache = st["k"], st["cache"]
    s, p = _token_rows(st["cu"], k.shape[0])
    pos = p + (st["lens"].long() - st["cu"].diff().long())[s]
    page, slot = st["table"][s, pos // PAGE].long(), pos % PAGE
    ids, at = page.unique(return_inverse=True)
    part = _codes(cache[ids])  # (the codes beside the new ones stay)
    for whole, x in zip(part, (*_quantise(k), *_quantise(st["v"]))):
        whole[at, slot] = x
    cache[ids] = _pack(*(x.flatten(0, 1) for x in part))
    if st["weights"] is not None:
        st["weights"][page, :, slot] = 0.0
    kc, ks, kl, vc, vs, vl = (x[at, slot] for x in _codes(cache[ids]))
    return {"k": _values(kc, ks, kl).to(k.dtype), "v": _values(vc, vs, vl).to(k.dtype), "weights": st["weights"]}


def _plain_decode(st):
    q, table, lens = st["q"], st["table"].long(), st["lens"].long()
    S = q.shape[1]
    kc, ks, kl, vc, vs, vl = _codes(st["cache"][table])
    k, v = _values(kc, ks, kl).flatten(1, 2), _values(vc, vs, vl).flatten(1, 2)
    limit = lens[:, None] - S + 1 + torch.arange(S, device=q.device)
    p, o = _attend(q.float(), k, v, limit, st["scale"])
    if st["weights"] is not None:
        B, H = len(lens), k.shape[2]
        w = p.view(B, H, -1, p.shape[-1]).sum(2).view(B, H, -1, PAGE).transpose(1, 2)
        ids, rows, at = table[st["rows"], st["at"]], st["rows"], st["at"]
        st["weights"][ids] += w[rows, at]
    return {"out": o.to(q.dtype), "weights": st["weights"]}


def _plain_evict(st):
    case, table, lens = st["case"], st["table"].long(), st["lens"].long()
    cache, weights, rows, at = st["cache"], st["weights"], st["rows"], st["at"]
    budget, recent, H = case["budget"], case["recent"], case["hkv"]
    B, n = table.shape[0], table.shape[1] * PAGE
    pos = torch.arange(n, device=table.device)
    w = weights[table].permute(0, 2, 1, 3).reshape(B, H, n)
    rank = w.masked_fill((pos >= lens[:, None] - recent)[:, None], math.inf)
    rank = rank.masked_fill((pos >= lens[:, None])[:, None], -math.inf)
    most = min(budget, n)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :most].sort(-1).values
    short = (lens <= budget)[:, None, None]  # these stay as they are
    src = torch.where(short, pos[:most], kept)
    ids, inside = table[rows, at], pos[:most] < lens[:, None, None].clamp_max(budget)

    def moved(x):  # [B, H, n, ...]: the kept tokens to the front, the others where they were
        i = src.view(*src.shape, *[1] * (x.dim() - 3)).expand(*src.shape, *x.shape[3:])
        x = x.clone()
        x[:, :, :most] = torch.where(short.view(B, *[1] * (x.dim() - 1)), x[:, :, :most], x.gather(2, i))
        return x

    # [B, pages, 16, H, x] -> [B, H, n, x]
    part = [moved(x.flatten(1, 2).transpose(1, 2)).transpose(1, 2).unflatten(1, (-1, PAGE)) for x in _codes(cache[table])]
    cache[ids] = _pack(*(x[rows, at].flatten(0, 1) for x in part))
    weights[ids] = moved(w).view(B, H, -1, PAGE).transpose(1, 2)[rows, at]
    s, p = _token_rows(st["cu_kept"], st["kept"])
    kc, ks, kl, vc, vs, vl = (x.flatten(1, 2)[s, p] for x in part)
    dt = cache.dtype
    out = torch.full((B, H, budget), -1, dtype=torch.int32, device=table.device)
    out[..., :most] = src.masked_fill(~inside, -1).to(torch.int32)
    return {"lens": lens.clamp_max(budget).to(torch.int32), "kept": out, "k": _values(kc, ks, kl).to(dt),
            "v": _values(vc, vs, vl).to(dt), "weights": weights}


# --- from the definitions, in 64 bits ----------------------------------------------------


def _stored(st, b, n):
    """K and V [n, Hkv, D] that the records of sequence b hold, code by code, in float64."""
    case, dev = st["case"], st["cache"].device
    D = case["D"]
    t, d = torch.arange(n, device=dev)[:, None], torch.arange(D, device=dev)[None, :]
    slot, g, e = t % PAGE, d // 64, d % 64
    rec = st["cache"][st["table"][b].long()[torch.arange(n, device=dev) // PAGE]]
    raw = rec.contiguous().view(torch.uint8).long()  # [n, Hkv, 18 D]
    meta = rec[..., 8 * D:].double()
    j = e % 8
    nib_k = (((e // 16) * PAGE + slot) * (D // 64) + g) * 16 + (e % 16) // 8 * 8 + j // 2 + j % 2 * 4
    nib_v = 16 * D + (((slot // 4) * 16 + e // 4) * 4 + slot % 4) * (D // 32) * 2 + g * 4 + e % 4
    at = (slot * (D // 64) + g) * 2
    both = []
    for nib, first in ((nib_k, 0), (nib_v, D // 2)):
        i = nib[:, None, :].expand(n, case["hkv"], D)
        code = raw.gather(2, i // 2) >> (i % 2 * 4) & 15
        m = (at + first)[:, None, :].expand(n, case["hkv"], D)
        both.append(code.double() * meta.gather(2, m) + meta.gather(2, m + 1))
    return both


def _softmax_rows(q, k, v, scale):
    """One sequence, q [n, Hq, D] its last n tokens, k / v [m, Hkv, D], in float64."""
    n, m, G = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    seen = torch.arange(m, device=q.device)[None] <= torch.arange(m - n, m, device=q.device)[:, None]
    outs, ps = [], []
    for h in range(q.shape[1]):
        s = (q[:, h] @ k[:, h // G].t() * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1)
        outs.append(p @ v[:, h // G])
        ps.append(p.sum(0))
    return torch.stack(outs, 1), torch.stack(ps, 0).view(-1, G, m).sum(1)


def _nearest_codes(x):
    """The values that x [N, H, D] in float64 (of type dt) is stored as: by counting the borders below."""
    dt = x.dtype
    d = x.double().view(*x.shape[:2], -1, 64)
    least = d.min(-1, keepdim=True).values
    s = ((d.max(-1, keepdim=True).values - least) / 15).float().to(dt).double()
    code = torch.zeros_like(d)
    for j in range(15):
        border = (2 * j + 1) * s
        twice = 2 * (d - least)
        code += (twice > border) | ((twice == border) & (j % 2 == 1))
    return (torch.where(s > 0, code, torch.zeros_like(code)) * s + least).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    new, total = st["new"], st["total"]
    op = case["op"]
    if op == "prompt":
        outs, a, b = [], 0, 0
        for n, m in zip(new, total):
            q, k, v = st["q"][a:a + n].double(), st["k"][b:b + m].double(), st["v"][b:b + m].double()
            outs.append(_softmax_rows(q, k, v, st["scale"])[0])
            a, b = a + n, b + m
        return torch.cat(outs)
    if op == "store":
        weights = None
        if st["weights"] is not None:
            weights = st["weights"].double()
            for s, t in enumerate(total):
                weights[st["table"][s, (t - 1) // PAGE].long(), :, (t - 1) % PAGE] = 0.0
        return {"k": _nearest_codes(st["k"]), "v": _nearest_codes(st["v"]), "weights": weights}
    if op == "decode":
        weights = None if st["weights"] is None else st["weights"].double()
        outs = []
        for s, m in enumerate(total):
            k, v = _stored(st, s, m)
            o, w = _softmax_rows(st["q"][s].double(), k, v, st["scale"])
            outs.append(o)
            if weights is not None:
                t = torch.arange(m, device=k.device)
                weights[st["table"][s].long()[t // PAGE], :, t % PAGE] += w.t()
        return {"out": torch.stack(outs), "weights": weights}
    budget, recent = case["budget"], case["recent"]
    weights = st["weights"].double()
    ks, vs = [], []
    kept = torch.full((len(total), case["hkv"], budget), -1, dtype=torch.int64)
    for s, m in enumerate(total):
        k, v = _stored(st, s, m)
        t = torch.arange(m, device=k.device)
        page, slot = st["table"][s].long()[t // PAGE], t % PAGE
        w = weights[page, :, slot]
        n = min(m, budget)
        if m <= budget:
            kept[s, :, :m] = torch.arange(m)
            ks.append(k)
            vs.append(v)
            continue
        old = w[:m - recent].cpu()
        for h in range(case["hkv"]):
            first = sorted(range(m - recent), key=lambda i, c=old[:, h].tolist(): (-c[i], i))[:n - recent]
            keep = torch.tensor(sorted(first) + list(range(m - recent, m)))
            kept[s, h, :n] = keep
            keep = keep.to(k.device)
            k[:n, h], v[:n, h], w[:n, h] = k[keep, h], v[keep, h], w[keep, h]
        ks.append(k[:n])
        vs.append(v[:n])
        weights[page, :, slot] = w
    lens = torch.tensor([min(m, budget) for m in total])
    return {"lens": lens, "kept": kept, "k": torch.cat(ks), "v": torch.cat(vs), "weights": weights}
