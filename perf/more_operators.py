"""Timed cases of the operators of a step with drafted token trees.

* ``rope``: a step's keys rotated by their positions and written to the
  quantized cache with the values, its queries rotated (``rope_kv_store_paged``).
* ``tree``: attention of a tree of drafted tokens over the cache, each token
  seeing the context and its own branch (``int8k_int4v_attn_tree``).
* ``logprobs``: log probabilities, ranks, entropies and likeliest tokens of
  rows of logits (``token_logprobs``).
* ``accept``: the branch of a drafted tree that the target model's tokens
  confirm (``accept_tree``).
* ``keep``: the cache rows of that branch moved to the places of a linear
  sequence (``kv_keep_paged``).

``run`` computes them with elementary torch operations in 32 bits (64 for the
keys' and queries' rounding rules and the positions' angles behind them), or,
where ``own`` is set, calls the op table.  ``exact`` restates them in 64 bits.
Cached rows come back dequantized, by ``kv_load_paged`` where ``own`` is set.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

PAGE = 64
GQA = 6  # query heads of a KV head
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One token of one request, as in a decode step: latency.
        _rope("rope_1_token", 4, 128, "fp16", "131071", "1", rot=128, table="fp32", neox=True, bound=True),
        # A step of eleven prompt chunks with some padding behind them.
        _rope("rope_11_chunks", 4, 128, "bf16", "0 0 0 512 4224 100 77 0 33000 1 640",
              "4224 4224 2112 2048 1000 1500 333 64 511 7 200", rot=128, table="bf16", neox=True),
        # One request, a small tree over a short context: latency.
        _tree("tree_1x13_over_2048", 4, 128, "fp16", 13, "2048", bound=True),
        # A serving batch at head dim 256 on a two-head rank, manager blocks of 33
        # pages, a tree of 26 nodes; one request is padding, one begins with its tree.
        _tree("tree_12x26_d256", 2, 256, "bf16", 26, "12000 0 8011 4097 -1 9000 15000 64 2300 6001 31 20000", ppb=33),
        # Large trees over long documents.
        _tree("tree_4x64_over_131072", 4, 128, "bf16", 64, "131072 130001 127 100000"),
        # The greedy token of one request with its alternatives: latency.
        _logprobs("logprobs_1x32000", 1, 32000, "fp32", 8, "plain", bound=True),
        # The nodes of a few trees, half of the rows under a grammar's mask.
        _logprobs("logprobs_48x65537_odd", 48, 65537, "fp16", 5, "masked"),
        # A prompt's log probabilities over a large vocabulary.
        _logprobs("logprobs_2048x152000", 2048, 152000, "bf16", 20, "plain"),
        # One request's tree, and a large batch's.
        _accept("accept_1x13", 1, 13, 6, bound=True),
        _accept("accept_256x64", 256, 64, 16),
        # The branch kept by one request, and by each of a large batch.
        _keep("keep_1x13", 4, 128, 13, "2048", bound=True),
        _keep("keep_128x26_d256", 2, 256, 26, " ".join(str(64 + (i * i * 977) % 3000) for i in range(128)), ppb=33),
    ]


def draw(rng):
    kind = rng.choice(("rope", "tree", "tree", "logprobs", "accept", "keep"))
    if kind == "logprobs":
        vocab = _log_int(rng, 100, 152000)
        rows = _log_int(rng, 1, min(4096, 2048 * 152000 // vocab))
        return _logprobs(None, rows, vocab, rng.choice(("fp32", "fp16", "bf16")), rng.choice((0, 1, 5, 20, rng.randint(1, 64))),
                         rng.choice(("plain", "masked")))
    nodes = _log_int(rng, 1, 64)
    if kind == "accept":
        return _accept(None, _log_int(rng, 1, 256), nodes, rng.randint(1, nodes))
    hkv, d, ppb = rng.choice((2, 4)), rng.choice((128, 256)), rng.choice((1, 1, 33))
    if kind == "rope":
        batch = _log_int(rng, 1, 64)
        most = 16384 * 128 * 4 // (d * hkv) // batch
        counts = [_log_int(rng, 1, max(1, most)) for _ in range(batch)]
        firsts = [rng.choice((0, _log_int(rng, 1, 4096))) for _ in range(batch)]
        rot = rng.choice((d, d, d // 2, d // 4, 16 * rng.randint(1, d // 16)))
        return _rope(None, hkv, d, rng.choice(("fp16", "bf16")), _text(firsts), _text(counts), rot=rot,
                     table=rng.choice(("fp32", "fp16", "bf16")), neox=rng.random() < 0.7, ppb=ppb)
    if kind == "keep":
        batch = _log_int(rng, 1, 128)
        return _keep(None, hkv, d, nodes, _text(_log_int(rng, 1, 4096) - 1 for _ in range(batch)), ppb=ppb)
    batch = _log_int(rng, 1, 64)
    # Scores and gathered rows (padded to the longest) stay below the largest listed case's.
    cap = 4 * 131072 * 4 * 128 // (hkv * d * batch)
    contexts = [-1 if rng.random() < 0.03 else _log_int(rng, 1, max(1, min(131072, cap))) - 1 for _ in range(batch)]
    return _tree(None, hkv, d, rng.choice(("fp16", "bf16")), nodes, _text(contexts), ppb=ppb)


def prepare(case, seed):
    kind = case["kind"]
    st = {"kind": kind, "case": case, **_inputs(case, seed)}
    if kind in ("rope", "keep"):
        n, dev = st["rows_to_read"], st["table"].device
        dt = torch.float32 if kind == "rope" else torch.float16
        st["k_out"] = torch.empty((n, case["hkv"], case["head_dim"]), dtype=dt, device=dev)
        st["v_out"] = torch.empty_like(st["k_out"])
    if kind == "rope":
        st["q_out"] = torch.empty(st["q"].shape, dtype=st["q"].dtype, device=st["q"].device)
    if kind == "tree":
        st["out"] = torch.empty(st["q"].shape, dtype=st["q"].dtype, device=st["q"].device)
    return st


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "tree": _plain_tree, "logprobs": _plain_logprobs, "accept": _plain_accept,
            "keep": _plain_keep}[state["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * (v * size + 8 + 4 + 4 + 4 + 12 * k), "flops": 4 * n * v}
    if kind == "accept":
        b, n, m = case["batch"], case["nodes"], case["width"]
        return {"bytes": b * (n * (4 + 4 + 8) + 12 * m + 12), "flops": b * n}
    hkv, d = case["hkv"], case["head_dim"]
    slot = d + d // 2 + 12  # cache bytes of one (token, KV head)
    if kind == "rope":
        # Rows in and out, a table row of cosines and sines a token, and the stored rows read back.
        n = sum(_ints(case["counts"]))
        tab = case["rot"] * (4 if case["table"] == "fp32" else 2)
        nbytes = n * (2 * GQA * hkv * d * 2 + 2 * hkv * d * 2 + 2 * hkv * slot + 16 + tab + 2 * hkv * d * 4)
        return {"bytes": nbytes, "flops": 3 * n * (GQA + 1) * hkv * case["rot"] + 6 * n * hkv * d}
    if kind == "keep":
        # Rows of an accepted branch (half a dozen) read and written; the tree's rows read back.
        n = len(_ints(case["contexts"]))
        kept = min(6, case["nodes"])
        return {"bytes": n * hkv * (2 * kept * slot + case["nodes"] * (slot + 4 * d)), "flops": 3 * n * case["nodes"] * hkv * d}
    n = case["nodes"]
    lens = [c + n if c >= 0 else 0 for c in _ints(case["contexts"])]
    nbytes = sum(lens) * hkv * slot + len(lens) * n * (2 * GQA * hkv * d * 2 + 8)
    return {"bytes": nbytes, "flops": 4 * d * GQA * hkv * sum(n * x for x in lens)}


def exact(case, seed):
    st = _inputs(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "logprobs": _exact_logprobs, "accept": _exact_accept,
            "keep": _exact_keep}[case["kind"]](case, st)


# ------------------------------------------------------------- the framework's calls
_OPS = []


def _table():
    if not _OPS:
        sys.path.insert(0, os.path.join(os.getcwd(), "k8v4-xpu_amd"))
        from k8v4_v030.ops_api import ops

        _OPS.append(ops())
    return _OPS[0]


def _run_own(st):
    o, case, kind = _table(), st["case"], st["kind"]
    if kind == "rope":
        _call(st, "call", o.bind_rope_kv_store_paged, o.rope_kv_store_paged,
              (st["q"], st["k"], st["v"], st["positions"], st["cos_sin"], case["neox"], st["slots"], *st["regions"],
               st["q_out"]))
        k, v = _read_back(o, st)
        return st["q_out"], k, v
    if kind == "keep":
        _call(st, "call", o.bind_kv_keep_paged, o.kv_keep_paged,
              (*st["regions"], st["table"], st["starts"], st["path"], st["accepted"], case["ppb"]))
        return _read_back(o, st)
    if kind == "tree":
        if "ws" not in st:  # the workspace, kept as a serving loop keeps it
            nbytes = o.attn_tree_workspace_bytes(st["lens"].shape[0], case["nodes"], case["hkv"], case["head_dim"])
            st["ws"] = torch.empty(-(-nbytes // 4), dtype=torch.int32, device=st["q"].device)
        _call(st, "call", o.bind_int8k_int4v_attn_tree, o.int8k_int4v_attn_tree,
              (st["q"], *st["regions"], st["table"], st["lens"], st["masks"], st["ws"], st["out"], case["nodes"],
               case["ppb"]))
        return st["out"]
    if kind == "accept":
        _call(st, "call", o.bind_accept_tree, o.accept_tree,
              (st["drafts"], st["parents"], st["targets"], st["lens"], st["path"], st["out_tokens"], st["accepted"],
               st["next_lens"]))
        return st["path"], st["out_tokens"], st["accepted"], st["next_lens"]
    if "ws" not in st:
        nbytes = o.token_logprobs_workspace_bytes(case["rows"], case["vocab"], case["top"])
        st["ws"] = torch.empty(max(4, -(-nbytes // 4)), dtype=torch.int32, device=st["logits"].device)
    _call(st, "call", o.bind_token_logprobs, o.token_logprobs,
          (st["logits"], st["tokens"], st["ws"], st["logprobs"], st["ranks"], st["entropy"], st["top_ids"],
           st["top_logprobs"]))
    return st["logprobs"], st["ranks"], st["entropy"], st["top_ids"], st["top_logprobs"]


def _read_back(o, st):
    _call(st, "load", o.bind_kv_load_paged, o.kv_load_paged,
          (*st["regions"], st["table"], st["starts"], st["rows"], st["case"]["ppb"], st["k_out"], st["v_out"]))
    return st["k_out"], st["v_out"]


def _call(st, name, bind, op, args):
    """The validating call, or (``bound``: a serving loop's) the call validated once."""
    if not st["case"]["bound"]:
        op(*args)
        return
    if name not in st:
        st[name] = bind(*args)
    st[name]()


# ---------------------------------------------------------------------- plain forms
def _over(x, n):
    """x / n, each quotient rounded once (by a Python number torch multiplies by its
    reciprocal, an ulp off, which moves codes that lie on a border)."""
    return x / torch.full_like(x, float(n))


def _dequantized(st, slots):
    """fp32 K and V ``[..., hkv, D]`` of the given cache slots."""
    k, ks, v, vs, vz = st["regions"]
    page, row = slots // PAGE, slots % PAGE
    kf = k[page, row].float() * ks[page, row][..., None]
    byte = v[page, row]
    nib = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).float()
    return kf, (nib - vz[page, row][..., None]) * vs[page, row][..., None]


def _slots(table, positions, ppb):
    """Cache slots of token positions through table rows (``[..., W]`` and ``[..., T]``)."""
    page = positions // PAGE
    entry = torch.gather(table, -1, page // ppb).long()
    return (entry * ppb + page % ppb) * PAGE + positions % PAGE


def _plain_read(st):
    """The rows that ``kv_load_paged`` gives."""
    rows, n = st["rows"].long(), st["rows_to_read"]
    b = torch.repeat_interleave(torch.arange(rows.shape[0] - 1, device=rows.device), rows[1:] - rows[:-1], output_size=n)
    pos = torch.arange(n, device=rows.device) - rows[b] + st["starts"].long()[b]
    page, ppb = pos // PAGE, st["case"]["ppb"]
    slots = (st["table"][b, page // ppb].long() * ppb + page % ppb) * PAGE + pos % PAGE
    k, v = _dequantized(st, slots)
    return k.to(st["k_out"].dtype), v.to(st["v_out"].dtype)


def _rotated(x, cos, sin, neox):
    """``[T, H, D]`` with the first ``2 * cos.shape[-1]`` dims of every head rotated."""
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    rot, rest = x[..., : 2 * half], x[..., 2 * half :]
    a, b = (rot[..., :half], rot[..., half:]) if neox else (rot[..., 0::2], rot[..., 1::2])
    first, second = a * c - b * s, b * c + a * s
    rot = torch.cat((first, second), -1) if neox else torch.stack((first, second), -1).flatten(-2)
    return torch.cat((rot, rest), -1)


def _plain_rope(st):
    case, q = st["case"], st["q"]
    angles = st["cos_sin"][st["positions"]]
    half = case["rot"] // 2
    cos, sin = angles[:, :half], angles[:, half:]
    q_out = _rotated(q.float(), cos.float(), sin.float(), case["neox"]).to(q.dtype)
    # The cache's rules in 64 bits: K symmetric int8, half away from zero; V affine uint4.
    k = _rotated(st["k"].double(), cos.double(), sin.double(), case["neox"])
    ks = _over(k.abs().amax(-1), 127)
    inv = torch.where(ks == 0, torch.zeros_like(ks), 1.0 / ks)[..., None]
    kc = (torch.sign(k) * torch.floor(k.abs() * inv + 0.5)).clamp(-127, 127).to(torch.int8)
    v = st["v"].double()
    lo = v.amin(-1)
    vs = _over(v.amax(-1) - lo, 15).clamp_min(1.0e-8)
    vz = torch.floor(-lo / vs + 0.5).clamp(0.0, 15.0)
    vc = torch.floor(v / vs[..., None] + vz[..., None] + 0.5).clamp(0.0, 15.0).to(torch.uint8)
    # Padding goes to a page that no sequence holds.
    kr, ksr, vr, vsr, vzr = st["regions"]
    slots = torch.where(st["slots"] < 0, torch.full_like(st["slots"], kr.shape[0] * PAGE - 1), st["slots"])
    page, row = slots // PAGE, slots % PAGE
    kr[page, row] = kc
    ksr[page, row] = ks.float()
    vr[page, row] = vc[..., 0::2] | (vc[..., 1::2] << 4)
    vsr[page, row] = vs.float()
    vzr[page, row] = vz.float()
    k_rows, v_rows = _plain_read(st)
    return q_out, k_rows, v_rows


def _plain_tree(st):
    case, q, lens = st["case"], st["q"], st["lens"].long()
    hkv, d, n, ppb = case["hkv"], case["head_dim"], case["nodes"], case["ppb"]
    batch, dev = lens.shape[0], q.device
    # The query row's int8 rule (half away from zero, in 64 bits).
    x = q.double()
    scale = _over(x.abs().amax(-1, keepdim=True), 127)
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    code = torch.sign(x) * torch.floor(x.abs() * inv + 0.5)
    rows = (code.float() * (scale.float() / math.sqrt(d))).view(batch, n, hkv, GQA, d)
    rows = rows.permute(0, 2, 1, 3, 4).reshape(batch * hkv, n * GQA, d)

    most = max(1, max(_ints(case["contexts"])) + n)
    t = torch.arange(most, device=dev)
    last = st["table"].shape[1] * ppb * PAGE - 1
    k, v = _dequantized(st, _slots(st["table"], t.clamp(max=last).expand(batch, most), ppb))
    k = k.permute(0, 2, 3, 1).reshape(batch * hkv, d, most)
    v = v.transpose(1, 2).reshape(batch * hkv, most, d)
    # A node sees the context, and of the tree what its mask holds.
    node = t[None, :] - (lens - n)[:, None]  # [batch, tokens]
    bit = (st["masks"][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
    seen = (node[:, None, :] < 0) | ((bit != 0) & (node < n)[:, None, :])  # [batch, nodes, tokens]
    seen = seen & (t[None, :] < lens[:, None])[:, None, :]
    s = torch.bmm(rows, k).view(batch, hkv, n * GQA, most)
    s.masked_fill_(~seen.repeat_interleave(GQA, 1)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(batch * hkv, n * GQA, most), v).view(batch, hkv, n * GQA, d)
    o = o / torch.where(total == 0, torch.ones_like(total), total)  # a row that sees nothing gives zeros
    o = o.view(batch, hkv, n, GQA, d).transpose(1, 2)
    return o.reshape(q.shape).to(q.dtype)


def _plain_logprobs(st):
    logits, tokens, k = st["logits"], st["tokens"], st["case"]["top"]
    x = logits.float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    vocab = x.shape[1]
    m = x.amax(-1, keepdim=True)
    some = m > -math.inf
    y = x - torch.where(some, m, torch.zeros_like(m))
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    log_total = torch.where(some, total.log(), torch.zeros_like(total))
    mean = torch.where(e > 0, y * e, torch.zeros_like(e)).sum(-1, keepdim=True) / torch.where(some, total, torch.ones_like(total))
    entropy = torch.where(some, log_total - mean, torch.zeros_like(mean))[:, 0]
    inside = (tokens >= 0) & (tokens < vocab)
    at = tokens.clamp(0, vocab - 1)[:, None]
    xt = torch.gather(x, 1, at)
    there = inside[:, None] & (xt > -math.inf)
    lp = torch.where(there, torch.gather(y, 1, at) - log_total, torch.full_like(xt, -math.inf))[:, 0]
    index = torch.arange(vocab, device=x.device)[None, :]
    ahead = ((x > xt) | ((x == xt) & (index < at))).sum(-1)
    rank = torch.where(there[:, 0], ahead + 1, torch.zeros_like(ahead)).to(torch.int32)
    # Ordered by value, then by lowest index: one key of both.
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 24) + (vocab - 1 - index)
    got = key.topk(min(k, vocab), dim=-1).values
    ids = vocab - 1 - (got & ((1 << 24) - 1))
    lps = torch.gather(y, 1, ids) - log_total
    live = torch.gather(x, 1, ids) > -math.inf
    ids = torch.where(live, ids, torch.full_like(ids, -1))
    lps = torch.where(live, lps, torch.full_like(lps, -math.inf))
    pad = (0, k - ids.shape[1])
    return (lp, rank, entropy, torch.nn.functional.pad(ids, pad, value=-1),
            torch.nn.functional.pad(lps, pad, value=-math.inf))


def _plain_accept(st):
    drafts, parents, targets = st["drafts"].long(), st["parents"].long(), st["targets"]
    n, m, dev = drafts.shape[1], st["case"]["width"], drafts.device
    i = torch.arange(n, device=dev)
    up = parents.clamp(min=0)
    fits = (drafts == torch.gather(targets, 1, up)) & (parents >= 0) & (parents < i)
    # Of siblings that fit, the first.
    twin = (parents[:, :, None] == parents[:, None, :]) & fits[:, None, :] & (i[None, :] < i[:, None])[None]
    link = fits & ~twin.any(-1)
    link[:, 0] = True
    # Ancestors: powers of "itself or its parent", seven doublings reach 128 levels.
    reach = torch.eye(n, device=dev)[None] + torch.nn.functional.one_hot(up, n).float() * (parents >= 0)[..., None]
    for _ in range(7):
        reach = torch.bmm(reach, reach).clamp_(max=1.0)
    on = (torch.bmm(reach, (~link).float()[..., None])[..., 0] == 0) & (reach[:, :, 0] > 0)
    place = on.long().cumsum(1) - 1
    on &= place < m
    count = on.sum(1)
    place = torch.where(on, place, torch.full_like(place, m))
    path = torch.full((drafts.shape[0], m + 1), -1, dtype=torch.int64, device=dev)
    path.scatter_(1, place, torch.where(on, i.expand_as(on), torch.full_like(place, -1)))
    path = path[:, :m]
    out = torch.where(path >= 0, torch.gather(targets, 1, path.clamp(min=0)), path)
    return path.to(torch.int32), out, (count - 1).to(torch.int32), (st["lens"] + count).to(torch.int32)


def _plain_keep(st):
    case, path = st["case"], st["path"].long()
    m, ppb, dev = path.shape[1], case["ppb"], path.device
    i = torch.arange(m, device=dev)
    moves = (i <= st["accepted"].long()[:, None]) & (path > i)
    base = st["starts"].long()[:, None]
    src = _slots(st["table"], base + torch.where(moves, path, i), ppb)
    dst = _slots(st["table"], base + i, ppb)
    spare = st["regions"][0].shape[0] * PAGE - 1  # of a page that no sequence holds
    src = torch.where(moves, src, torch.full_like(src, spare)).flatten()
    dst = torch.where(moves, dst, torch.full_like(dst, spare)).flatten()
    rows = [x[src // PAGE, src % PAGE] for x in st["regions"]]
    for x, row in zip(st["regions"], rows):
        x[dst // PAGE, dst % PAGE] = row
    return _plain_read(st)


# ----------------------------------------------------------------- 64-bit restatements
def _whole_rows(regions, slots):
    """float64 K and V rows of slots."""
    k, ks, v, vs, vz = regions
    p, r = torch.div(slots, PAGE, rounding_mode="floor"), slots.remainder(PAGE)
    kd = k[p, r].double()
    kd *= ks[p, r].double().unsqueeze(-1)
    packed = v[p, r].int()
    vd = torch.empty_like(kd)
    vd[..., 0::2] = (packed % 16).double()
    vd[..., 1::2] = torch.div(packed, 16, rounding_mode="floor").double()
    vd -= vz[p, r].double().unsqueeze(-1)
    vd *= vs[p, r].double().unsqueeze(-1)
    return kd, vd


def _row_slots(row, first, count, ppb):
    pos = torch.arange(first, first + count, device=row.device)
    blk = torch.div(pos, PAGE * ppb, rounding_mode="floor")
    return row[blk].long() * (PAGE * ppb) + pos.remainder(PAGE * ppb)


def _turned(x, angles, neox):
    """Rotation as a complex product, in 64 bits."""
    half = angles.shape[-1] // 2
    w = torch.complex(angles[:, None, :half].double(), angles[:, None, half:].double())
    y = x.double().clone()
    a, b = (slice(0, half), slice(half, 2 * half)) if neox else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(y[..., a].clone(), y[..., b].clone()) * w
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_rope(case, st):
    n = st["rows_to_read"]
    angles = st["cos_sin"][st["positions"]]
    q = _turned(st["q"], angles, case["neox"])
    k = _turned(st["k"], angles, case["neox"])[:n]  # padding lies behind the step's tokens
    step = _over(k.abs().amax(-1, keepdim=True), 127)
    y = k * torch.where(step == 0, torch.zeros_like(step), 1.0 / step)
    code = torch.where(y >= 0, torch.floor(y + 0.5), torch.ceil(y - 0.5))
    v = st["v"][:n].double()
    low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    unit = torch.clamp(_over(high - low, 15), min=1.0e-8)
    zero = torch.clamp(torch.floor(-low / unit + 0.5), 0, 15)
    nib = torch.clamp(torch.floor(v / unit + zero + 0.5), 0, 15)
    return q, code * step.float().double(), (nib - zero) * unit.float().double()


def _exact_tree(case, st):
    hkv, d, n, ppb = case["hkv"], case["head_dim"], case["nodes"], case["ppb"]
    q = st["q"].double()
    amax = q.abs().amax(-1)
    step = torch.where(amax == 0, torch.ones_like(amax), _over(amax, 127))
    y = q * (1.0 / step)[..., None]
    q = torch.where(y >= 0, torch.floor(y + 0.5), torch.ceil(y - 0.5)) * step[..., None]
    out = torch.zeros_like(q)
    for b, context in enumerate(_ints(case["contexts"])):
        if context < 0:
            continue
        keys, values = _whole_rows(st["regions"], _row_slots(st["table"][b], 0, context + n, ppb))
        hidden = torch.zeros((n, context + n), dtype=torch.bool, device=q.device)
        words = st["masks"][b].tolist()
        hidden[:, context:] = torch.tensor([[(w >> j) & 1 == 0 for j in range(n)] for w in words], device=q.device)
        hidden = hidden.repeat_interleave(GQA, 0)
        for h in range(hkv):
            rows = q[b * n : (b + 1) * n, GQA * h : GQA * (h + 1)].reshape(-1, d)
            s = torch.mm(rows, keys[:, h].t()) / math.sqrt(d)
            p = torch.softmax(s.masked_fill_(hidden, -math.inf), dim=1).nan_to_num_(0.0)
            out[b * n : (b + 1) * n, GQA * h : GQA * (h + 1)] = torch.mm(p, values[:, h]).view(n, GQA, d)
    return out


def _exact_logprobs(case, st):
    got = ([], [], [], [], [])
    k = case["top"]
    for lo in range(0, case["rows"], 64):
        x = st["logits"][lo : lo + 64].double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        t = st["tokens"][lo : lo + 64]
        lp = torch.log_softmax(x, -1)
        lp = torch.where(torch.isnan(lp), torch.full_like(lp, -math.inf), lp)
        p = lp.exp()
        inside = (t >= 0) & (t < x.shape[1])
        mine = torch.where(inside, lp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0], torch.full_like(lp[:, 0], -math.inf))
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        place = (order == t[:, None]).int().argmax(-1) + 1
        ids = torch.full((x.shape[0], k), -1, dtype=torch.int64, device=x.device)
        lps = torch.full((x.shape[0], k), -math.inf, dtype=torch.float64, device=x.device)
        w = min(k, x.shape[1])
        ids[:, :w], lps[:, :w] = order[:, :w], lp.gather(1, order[:, :w])
        ids[lps == -math.inf] = -1
        for out, value in zip(got, (mine, torch.where(mine > -math.inf, place, torch.zeros_like(place)).to(torch.int32),
                                    -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1), ids, lps)):
            out.append(value)
    return tuple(torch.cat(x) for x in got)


def _exact_accept(case, st):
    m, paths, outs = case["width"], [], []
    for drafts, parents, targets in zip(st["drafts"].tolist(), st["parents"].tolist(), st["targets"].tolist()):
        path = [0]
        while len(path) < m:
            children = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and drafts[i] == targets[path[-1]]]
            if not children:
                break
            path.append(children[0])
        paths.append(path + [-1] * (m - len(path)))
        outs.append([targets[i] for i in path] + [-1] * (m - len(path)))
    path = torch.tensor(paths, dtype=torch.int32, device=st["drafts"].device)
    count = (path >= 0).sum(1).to(torch.int32)
    return path, torch.tensor(outs, device=path.device), count - 1, st["lens"] + count


def _exact_keep(case, st):
    ks, vs = [], []
    for b, base in enumerate(_ints(case["contexts"])):
        k, v = _whole_rows(st["regions"], _row_slots(st["table"][b], base, case["nodes"], case["ppb"]))
        kept_k, kept_v = k.clone(), v.clone()
        for i, node in enumerate(st["path"][b].tolist()[: int(st["accepted"][b]) + 1]):
            kept_k[i], kept_v[i] = k[node], v[node]
        ks.append(kept_k)
        vs.append(kept_v)
    return torch.cat(ks), torch.cat(vs)


# ------------------------------------------------------------------------------ inputs
def _named(name, case):
    return case if name is None else {"name": name, **case}


def _rope(name, hkv, head_dim, dtype, firsts, counts, rot, table, neox, ppb=1, bound=False):
    """``counts`` tokens of each sequence from position ``firsts`` on; the first ``rot`` dims rotate."""
    return _named(name, {"kind": "rope", "hkv": hkv, "head_dim": head_dim, "dtype": dtype, "firsts": firsts,
                         "counts": counts, "rot": rot, "table": table, "neox": neox, "ppb": ppb, "bound": bound})


def _tree(name, hkv, head_dim, dtype, nodes, contexts, ppb=1, bound=False):
    """``contexts``: cached tokens ahead of each sequence's tree (-1: a padding request without tokens)."""
    return _named(name, {"kind": "tree", "hkv": hkv, "head_dim": head_dim, "dtype": dtype, "nodes": nodes,
                         "contexts": contexts, "ppb": ppb, "bound": bound})


def _logprobs(name, rows, vocab, dtype, top, rows_are, bound=False):
    return _named(name, {"kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
                         "rows_are": rows_are, "bound": bound})


def _accept(name, batch, nodes, width, bound=False):
    """``width``: the longest branch that is followed, the root included."""
    return _named(name, {"kind": "accept", "batch": batch, "nodes": nodes, "width": width, "bound": bound})


def _keep(name, hkv, head_dim, nodes, contexts, ppb=1, bound=False):
    return _named(name, {"kind": "keep", "hkv": hkv, "head_dim": head_dim, "nodes": nodes, "contexts": contexts,
                         "ppb": ppb, "bound": bound})


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def _text(values):
    return " ".join(str(int(x)) for x in values)


def _ints(text):
    return [int(x) for x in text.split()]


def _generator(seed, what):
    return torch.Generator(device="cuda" if torch.cuda.is_available() else "cpu").manual_seed(1000003 * seed + what)


def _inputs(case, seed):
    return {"rope": _rope_inputs, "tree": _tree_inputs, "logprobs": _logit_inputs, "accept": _accept_inputs,
            "keep": _keep_inputs}[case["kind"]](case, seed)


def _cache(case, seed, lens):
    """A pool of region-major pages, its five views, and the block table of
    sequences of ``lens`` tokens at random physical blocks; the pool's last block
    belongs to none.  K rows are int8 codes of channels of uneven size (as rotary
    keys have) with a scale a row, V rows uint4 codes with a scale and a zero
    point a row."""
    hkv, d, ppb = case["hkv"], case["head_dim"], case["ppb"]
    gen = _generator(seed, 1)
    dev = gen.device
    need = [-(-n // (PAGE * ppb)) for n in lens]
    pool = sum(need) + sum(need) // 10 + 2
    perm = torch.randperm(pool - 1, generator=torch.Generator().manual_seed(1000003 * seed + 2)).to(torch.int32)
    table = torch.zeros((len(lens), max(1, *need)) if len(need) > 1 else (1, max(1, need[0])), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at : at + n]
        at += n
    page_bytes = PAGE * hkv * (d + d // 2 + 12)
    raw = torch.empty((pool * ppb, page_bytes), dtype=torch.int8, device=dev)
    kb, vb, sb = PAGE * hkv * d, PAGE * hkv * d // 2, PAGE * hkv * 4
    channel = torch.exp(0.4 * torch.randn((hkv, d), generator=gen, device=dev))
    for lo in range(0, raw.shape[0], 512):
        part = raw[lo : lo + 512]
        n = part.shape[0]
        x = torch.randn((n, PAGE, hkv, d), generator=gen, device=dev) * channel
        amax = x.abs().amax(-1) / 127.0
        part[:, :kb] = torch.round(x / amax[..., None]).to(torch.int8).view(n, -1)
        part[:, kb : kb + vb] = torch.randint(-128, 128, (n, vb), generator=gen, device=dev, dtype=torch.int8)
        planes = torch.empty((n, 3, PAGE, hkv), device=dev)
        planes[:, 0] = amax
        planes[:, 1] = 0.3 + 0.1 * torch.rand((n, PAGE, hkv), generator=gen, device=dev)
        planes[:, 2] = torch.randint(5, 11, (n, PAGE, hkv), generator=gen, device=dev).float()
        part[:, kb + vb :] = planes.view(torch.int8).view(n, -1)
    flat = raw.view(-1)

    def view(dtype, size, start, inner):
        x = flat.view(dtype)
        strides = [1]
        for m in reversed(inner):
            strides.insert(0, strides[0] * m)
        return x.as_strided((raw.shape[0], *inner), (page_bytes // size, *strides[1:]), start // size)

    regions = (view(torch.int8, 1, 0, (PAGE, hkv, d)), view(torch.float32, 4, kb + vb, (PAGE, hkv)),
               view(torch.uint8, 1, kb, (PAGE, hkv, d // 2)), view(torch.float32, 4, kb + vb + sb, (PAGE, hkv)),
               view(torch.float32, 4, kb + vb + 2 * sb, (PAGE, hkv)))
    return {"raw": raw, "regions": regions, "table": table.to(dev)}


def _projected(case, tokens, seed):
    """Query, key and value views of a fused qkv projection's rows, as a model hands them over."""
    hkv, d = case["hkv"], case["head_dim"]
    gen = _generator(seed, 3)
    buf = (0.5 * torch.randn((tokens, (GQA + 2) * hkv * d), generator=gen, device=gen.device)).to(_DTYPES[case["dtype"]])
    q, k, v = buf.split([GQA * hkv * d, hkv * d, hkv * d], 1)
    return q.unflatten(1, (GQA * hkv, d)), k.unflatten(1, (hkv, d)), v.unflatten(1, (hkv, d))


def _rope_inputs(case, seed):
    firsts, counts = _ints(case["firsts"]), _ints(case["counts"])
    st = _cache(case, seed, [f + n for f, n in zip(firsts, counts)])
    dev, n, ppb, half = st["table"].device, sum(counts), case["ppb"], case["rot"] // 2
    padded = n if case["bound"] else -(-n // 8) * 8  # a captured batch size
    st["q"], st["k"], st["v"] = _projected(case, padded, seed)
    st["starts"] = torch.tensor(firsts, dtype=torch.int32, device=dev)
    st["rows"] = torch.tensor([0, *counts]).cumsum(0).to(device=dev, dtype=torch.int32)
    st["rows_to_read"] = n
    pos, slots = torch.zeros(padded, dtype=torch.int64), torch.full((padded,), -1, dtype=torch.int64)
    at, table = 0, st["table"].cpu()
    for b, (first, count) in enumerate(zip(firsts, counts)):
        pos[at : at + count] = torch.arange(first, first + count)
        slots[at : at + count] = _row_slots(table[b], first, count, ppb)
        at += count
    st["positions"], st["slots"] = pos.to(dev), slots.to(dev)
    # A model's table of cosines and sines: base 10,000, up to the longest context, other seeds other bases.
    reach = max(f + c for f, c in zip(firsts, counts))
    inv = (10000.0 + seed % 97) ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
    angle = torch.arange(reach, dtype=torch.float64, device=dev)[:, None] * inv
    st["cos_sin"] = torch.cat((angle.cos(), angle.sin()), 1).to(_DTYPES[case["table"]])
    return st


def _trees(batch, nodes, seed):
    """Parents ``[batch, nodes]`` of random trees (a parent ahead of its children, -1: the root) and, as words, each
    node's branch."""
    gen = torch.Generator().manual_seed(1000003 * seed + 5)
    u = torch.rand((batch, nodes), generator=gen).maximum(torch.rand((batch, nodes), generator=gen))
    parents = (u * torch.arange(nodes)).to(torch.int32)
    parents[:, 0] = -1
    masks = torch.zeros((batch, nodes), dtype=torch.int64)
    one = torch.ones(1, dtype=torch.int64)
    masks[:, 0] = 1
    for i in range(1, nodes):
        masks[:, i] = masks.gather(1, parents[:, i : i + 1].long())[:, 0] | (one << i)
    return parents, masks


def _tree_inputs(case, seed):
    contexts, n = _ints(case["contexts"]), case["nodes"]
    lens = [c + n if c >= 0 else 0 for c in contexts]
    st = _cache(case, seed, lens)
    dev = st["table"].device
    st["q"], _k, _v = _projected(case, n * len(lens), seed)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["masks"] = _trees(len(lens), n, seed)[1].to(dev)
    return st


def _logit_inputs(case, seed):
    """A model's logits, some rows sure of one token; under ``masked`` half of the
    rows keep a few to a few hundred tokens, the others at minus infinity."""
    n, v, dt = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    gen = _generator(seed, 4)
    dev = gen.device
    logits = torch.empty((n, v), dtype=dt, device=dev)
    tokens = torch.empty((n,), dtype=torch.int64, device=dev)
    for lo in range(0, n, 64):
        x = 2.5 * torch.randn((min(64, n - lo), v), generator=gen, device=dev)
        m = x.shape[0]
        sure = torch.rand((m, 1), generator=gen, device=dev) < 0.3
        at = torch.randint(0, v, (m, 1), generator=gen, device=dev)
        x.scatter_add_(1, at, torch.where(sure, 22.0, 0.0))
        if case["rows_are"] == "masked":
            few = torch.rand((m, 1), generator=gen, device=dev) * torch.rand((m, 1), generator=gen, device=dev) * 300 / v
            keep = torch.rand((m, v), generator=gen, device=dev) < few
            keep |= torch.rand((m, 1), generator=gen, device=dev) < 0.5
            keep.scatter_(1, at, True)
            x.masked_fill_(~keep, -math.inf)
        logits[lo : lo + m] = x.to(dt)
        noise = torch.empty_like(x).exponential_(generator=gen)
        tokens[lo : lo + m] = (torch.softmax(x, -1) / noise).argmax(-1)
    k = case["top"]
    return {
        "logits": logits, "tokens": tokens,
        "logprobs": torch.empty((n,), device=dev), "entropy": torch.empty((n,), device=dev),
        "ranks": torch.empty((n,), dtype=torch.int32, device=dev),
        "top_ids": torch.empty((n, k), dtype=torch.int64, device=dev),
        "top_logprobs": torch.empty((n, k), device=dev),
    }


def _accept_inputs(case, seed):
    """Drafts of a small vocabulary's size, so that siblings differ, and for most
    inner nodes a target token that one of the children holds."""
    b, n, m = case["batch"], case["nodes"], case["width"]
    gen = torch.Generator().manual_seed(1000003 * seed + 6)
    parents, _masks = _trees(b, n, seed)
    drafts = torch.randint(0, 32000, (b, n), generator=gen, dtype=torch.int32)
    targets = torch.randint(0, 32000, (b, n), generator=gen)
    hit = torch.rand((b, n), generator=gen) < 0.6
    for i in range(1, n):
        up = parents[:, i : i + 1].long()
        new = torch.where(hit[:, i : i + 1], drafts[:, i : i + 1].long(), targets.gather(1, up))
        targets.scatter_(1, up, new)
    dev = _generator(seed, 7).device
    return {
        "drafts": drafts.to(dev), "parents": parents.to(dev), "targets": targets.to(dev),
        "lens": torch.randint(n, 100000, (b,), generator=gen, dtype=torch.int32).to(dev),
        "path": torch.empty((b, m), dtype=torch.int32, device=dev),
        "out_tokens": torch.empty((b, m), dtype=torch.int64, device=dev),
        "accepted": torch.empty((b,), dtype=torch.int32, device=dev),
        "next_lens": torch.empty((b,), dtype=torch.int32, device=dev),
    }


def _keep_inputs(case, seed):
    """Trees in the cache and the branch to the root of one node of each."""
    contexts, n = _ints(case["contexts"]), case["nodes"]
    st = _cache(case, seed, [c + n for c in contexts])
    dev, b = st["table"].device, len(contexts)
    _parents, masks = _trees(b, n, seed)
    gen = torch.Generator().manual_seed(1000003 * seed + 8)
    leaf = torch.randint(n // 2, n, (b, 1), generator=gen)
    bits = (masks.gather(1, leaf) >> torch.arange(n)) & 1
    order = torch.where(bits > 0, torch.arange(n), torch.full((b, n), n)).sort(1).values
    st["path"] = torch.where(order < n, order, torch.full_like(order, -1)).to(device=dev, dtype=torch.int32)
    st["accepted"] = (bits.sum(1) - 1).to(device=dev, dtype=torch.int32)
    st["starts"] = torch.tensor(contexts, dtype=torch.int32, device=dev)
    st["rows"] = (torch.arange(b + 1) * n).to(device=dev, dtype=torch.int32)
    st["rows_to_read"] = b * n
    return st
