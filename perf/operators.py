"""Timed cases of three operators around the quantized cache.

* ``shared``: one decode or MTP-verify step of a batch whose sequences begin
  with the same cached pages (``int8k_int4v_attn_shared``).
* ``load``: cached K/V rows of a ragged batch read back as fp16, bf16 or fp32
  (``kv_load_paged``).
* ``verify``: acceptance of drafted tokens against the target's probabilities
  and the token that follows them (``verify_drafts``).

``run`` computes them with elementary torch operations in 32 bits (64 for the
query's rounding rule, the acceptance test and the cumulative sums), or, where
``own`` is set, calls the op table.  ``exact`` restates them in 64 bits, one
sequence at a time.
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
        # A few requests behind a short system prompt, one token each: latency.
        _shared("shared_8_over_2048_q1", 4, 128, "fp16", 1, 2048, "1 17 40 64 90 128 200 300", bound=True),
        # A two-head rank at head dim 256, manager blocks of 33 pages, one
        # draft token, a prompt that does not end with a page; one request is
        # padding (no tokens at all).
        _shared("shared_24_over_8011_q2_d256", 2, 256, "bf16", 2, 8011,
                "2 93 214 377 640 701 1025 1100 1333 1590 1817 2048 2300 11 2 3 64 65 130 500 800 900 1000 0", ppb=33),
        # MTP verify of five continuations of a long document.
        _shared("shared_5_over_40000_q7", 4, 128, "bf16", 7, 40000, "7 100 555 1024 4100"),
        # Parallel sampling: 48 completions of one 128K-token document.
        _shared("shared_48_over_131072_q1", 4, 128, "bf16", 1, 131072,
                " ".join(str(20 + (i * i * 977) % 1700) for i in range(48))),
        # Parallel sampling with drafts: 64 completions, four tokens each.
        _shared("shared_64_over_100000_q4", 4, 128, "fp16", 4, 100000,
                " ".join(str(4 + (i * i * 631) % 1000) for i in range(64))),
        # One short sequence read back, as for a prompt moved to host memory.
        _load("load_1_of_500", 4, 128, "fp16", "0", "500", bound=True),
        # The tails of twelve sequences of a two-head rank at head dim 256,
        # each from another token on.
        _load("load_12_tails_d256", 2, 256, "bf16", "0 64 100 1000 33 7 0 2048 4000 5 63 65",
              "1 700 2500 64 65 1 0 900 3333 4096 129 8000", ppb=33),
        # Two long sequences for a transfer to another rank.
        _load("load_2_of_131072", 4, 128, "bf16", "0 0", "131072 131072"),
        # One request, three greedily drafted tokens.
        _verify("verify_1x3_greedy", 1, 3, 32000, "fp32", drafts="greedy", filtered=False, bound=True),
        # A serving batch with ragged draft counts, 16-bit probabilities and an
        # odd vocabulary.
        _verify("verify_48x6_odd", 48, 6, 65537, "bf16", drafts="sampled", filtered=True),
        # A large batch over a large vocabulary.
        _verify("verify_256x4", 256, 4, 152000, "fp32", drafts="sampled", filtered=False),
    ]


def draw(rng):
    kind = rng.choice(("shared", "shared", "load", "verify"))
    if kind == "verify":
        vocab, batch, drafts = _log_int(rng, 1000, 152000), _log_int(rng, 1, 256), rng.randint(1, 9)
        batch = max(1, min(batch, 256 * 5 * 152000 // (vocab * (drafts + 1))))
        return _verify(None, batch, drafts, vocab, rng.choice(("fp32", "fp16", "bf16")),
                       drafts=rng.choice(("sampled", "sampled", "greedy")), filtered=rng.random() < 0.5)
    hkv, d, ppb = rng.choice((2, 4)), rng.choice((128, 256)), rng.choice((1, 1, 33))
    if kind == "load":
        batch = _log_int(rng, 1, 64)
        budget = 262144 * 128 // d * 4 // hkv // 2
        counts = [_log_int(rng, 1, max(1, budget // batch)) - 1 for _ in range(batch)]
        firsts = [rng.choice((0, _log_int(rng, 1, 4096))) for _ in range(batch)]
        return _load(None, hkv, d, rng.choice(("fp16", "bf16", "fp32")), _text(firsts), _text(counts), ppb=ppb)
    q_len, batch = rng.choice((1, 1, 2, 4, 7, rng.randint(1, 10))), _log_int(rng, 2, 64)
    # Scores of the prefix and gathered suffix rows stay below the largest listed case's.
    prefix = _log_int(rng, 64, min(131072, 64 * 4 * 100000 * 4 * 128 // (hkv * d * batch * q_len)))
    top = min(4096, max(q_len + 1, 48 * 1700 * 4 * 128 // (hkv * d * batch)))
    own_tokens = [0 if rng.random() < 0.03 else _log_int(rng, q_len, top) for _ in range(batch)]
    return _shared(None, hkv, d, rng.choice(("fp16", "bf16")), q_len, prefix, _text(own_tokens), ppb=ppb)


def prepare(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return {"kind": kind, "case": case, **_drafted(case, seed)}
    cache = _cache(case, seed)
    st = {"kind": kind, "case": case, **cache}
    dt, dev = _DTYPES[case["dtype"]], cache["raw"].device
    hkv, d = case["hkv"], case["head_dim"]
    if kind == "load":
        counts = _ints(case["counts"])
        starts = torch.tensor([0, *counts], dtype=torch.int64).cumsum(0)
        st["firsts"] = torch.tensor(_ints(case["firsts"]), dtype=torch.int32, device=dev)
        st["rows"] = starts.to(device=dev, dtype=torch.int32)
        shape = (sum(counts), hkv, d)
        st["k_out"], st["v_out"] = torch.empty(shape, dtype=dt, device=dev), torch.empty(shape, dtype=dt, device=dev)
        return st
    st["q"] = _queries(case, seed)
    st["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    st["out"] = torch.empty(st["q"].shape, dtype=dt, device=dev)
    return st


def run(state):
    if own:
        return _run_own(state)
    return {"shared": _plain_shared, "load": _plain_load, "verify": _plain_verify}[state["kind"]](state)


def work(case):
    kind = case["kind"]
    if kind == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        rows = 1 if case["how"] == "greedy" else 2  # a row of the target, and one of the draft
        return {"bytes": b * (rows * v * size + k * (8 + 2 * size) + 8 * (k + 1) + 20), "flops": 2 * b * rows * v}
    hkv, d = case["hkv"], case["head_dim"]
    slot = d + d // 2 + 12  # cache bytes of one (token, KV head)
    if kind == "load":
        n = sum(_ints(case["counts"]))
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * hkv * (slot + 2 * d * size), "flops": 3 * n * hkv * d}
    lens, q_len = _lengths(case), case["q_len"]
    tokens = case["prefix"] + sum(max(0, n - case["prefix"]) for n in lens)
    pairs = sum(max(0, n - q_len + j + 1) for n in lens for j in range(q_len))
    nbytes = tokens * hkv * slot + 2 * len(lens) * q_len * GQA * hkv * d * 2
    return {"bytes": nbytes, "flops": 4 * d * GQA * hkv * pairs}


def exact(case, seed):
    if case["kind"] == "verify":
        return _exact_verify(case, _drafted(case, seed))
    cache = _cache(case, seed)
    if case["kind"] == "load":
        return _exact_load(case, cache)
    return _exact_shared(case, cache, _queries(case, seed))


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
    if kind == "shared":
        q = st["q"]
        if "ws" not in st:  # the workspace, kept as a serving loop keeps it
            nbytes = o.attn_shared_workspace_bytes(q.shape[0] // case["q_len"], case["q_len"], case["hkv"],
                                                   case["head_dim"])
            st["ws"] = torch.empty(-(-nbytes // 4), dtype=torch.int32, device=q.device)
        args = (q, *st["regions"], st["prefix_table"], case["prefix"], st["table"], st["lens"], st["ws"], st["out"],
                case["q_len"], case["ppb"])
        _call(st, o.bind_int8k_int4v_attn_shared, o.int8k_int4v_attn_shared, args)
        return st["out"]
    if kind == "load":
        args = (*st["regions"], st["table"], st["firsts"], st["rows"], case["ppb"], st["k_out"], st["v_out"])
        _call(st, o.bind_kv_load_paged, o.kv_load_paged, args)
        return st["k_out"], st["v_out"]
    if "ws" not in st:
        nbytes = o.verify_drafts_workspace_bytes(case["batch"], case["vocab"])
        st["ws"] = torch.empty(-(-nbytes // 4), dtype=torch.int32, device=st["target"].device)
    args = (st["target"], st["draft"], st["tokens"], st["counts"], st["accept_u"], st["sample_u"], st["lens"],
            st["ws"], st["out_tokens"], st["accepted"], st["next_lens"])
    _call(st, o.bind_verify_drafts, o.verify_drafts, args)
    return st["out_tokens"], st["accepted"], st["next_lens"]


def _call(st, bind, op, args):
    """The validating call, or (``bound``: a serving loop's) the call validated once."""
    if not st["case"]["bound"]:
        op(*args)
        return
    if "call" not in st:
        st["call"] = bind(*args)
    st["call"]()


# ---------------------------------------------------------------------- plain forms
def _dequantized(st, slots):
    """fp32 K and V ``[..., hkv, D]`` of the given cache slots."""
    k, ks, v, vs, vz = st["regions"]
    page, row = slots // PAGE, slots % PAGE
    kf = k[page, row].float() * ks[page, row][..., None]
    byte = v[page, row]
    nib = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).float()
    return kf, (nib - vz[page, row][..., None]) * vs[page, row][..., None]


def _slots(row, positions, ppb):
    """Cache slots of token positions through table rows (``row`` as long as ``positions`` in its leading dims)."""
    page = positions // PAGE
    entry = torch.gather(row, -1, page // ppb).long()
    return (entry * ppb + page % ppb) * PAGE + positions % PAGE


def _plain_load(st):
    table, rows, firsts, ppb = st["table"], st["rows"].long(), st["firsts"].long(), st["case"]["ppb"]
    counts = rows[1:] - rows[:-1]
    n = st["k_out"].shape[0]
    b = torch.repeat_interleave(torch.arange(table.shape[0], device=table.device), counts, output_size=n)
    pos = torch.arange(n, device=table.device) - rows[b] + firsts[b]
    page = pos // PAGE
    slots = (table[b, page // ppb].long() * ppb + page % ppb) * PAGE + pos % PAGE
    k, v = _dequantized(st, slots)
    return k.to(st["k_out"].dtype), v.to(st["v_out"].dtype)


def _plain_shared(st):
    case, q = st["case"], st["q"]
    hkv, d, q_len, ppb = case["hkv"], case["head_dim"], case["q_len"], case["ppb"]
    batch, dev = q.shape[0] // q_len, q.device
    prefix = case["prefix"] // PAGE * PAGE  # whole pages are shared
    # The query row's int8 rule (half away from zero, in 64 bits).
    x = q.double()
    scale = x.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    code = torch.sign(x) * torch.floor(x.abs() * inv + 0.5)
    rows = (code.float() * (scale.float() / math.sqrt(d))).view(batch, q_len, hkv, GQA, d)
    ends = st["lens"].long()[:, None] - q_len + 1 + torch.arange(q_len, device=dev)  # [batch, q_len]

    # Scores over the prefix, [hkv, batch * q_len * 6, prefix], and over each
    # sequence's own tokens, [batch, hkv, q_len * 6, own].
    t = torch.arange(prefix, device=dev)
    kp, vp = _dequantized(st, _slots(st["prefix_table"], t, ppb))
    kp, vp = kp.permute(1, 2, 0).contiguous(), vp.transpose(0, 1).contiguous()
    sp = torch.bmm(rows.permute(2, 0, 1, 3, 4).reshape(hkv, -1, d), kp)
    sp.masked_fill_((t[None, :] >= ends.reshape(-1, 1).repeat_interleave(GQA, 0))[None], -math.inf)
    most = max(1, max(_lengths(case)) - prefix)
    t = (prefix + torch.arange(most, device=dev)).clamp(max=st["table"].shape[1] * ppb * PAGE - 1)
    seen = (prefix + torch.arange(most, device=dev))[None, None, :] < ends[:, :, None]  # [batch, q_len, own]
    ks, vs = _dequantized(st, _slots(st["table"], t.expand(batch, most), ppb))
    ks, vs = ks.permute(0, 2, 3, 1).reshape(batch * hkv, d, most), vs.transpose(1, 2).reshape(batch * hkv, most, d)
    ss = torch.bmm(rows.transpose(1, 2).reshape(batch * hkv, q_len * GQA, d), ks)
    hidden = ~seen[:, None].repeat_interleave(GQA, 2)  # [batch, 1, q_len * 6, own]
    ss = ss.view(batch, hkv, q_len * GQA, most).masked_fill_(hidden, -math.inf)

    # One softmax over both; a row that sees nothing gives zeros.
    top = ss.amax(-1)
    if prefix:
        top = torch.maximum(top, sp.amax(-1).view(hkv, batch, q_len * GQA).transpose(0, 1))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    pp = sp.sub_(top.transpose(0, 1).reshape(hkv, -1, 1)).exp_()
    ps = ss.sub_(top[..., None]).exp_()
    total = ps.sum(-1) + pp.sum(-1).view(hkv, batch, q_len * GQA).transpose(0, 1)
    o = torch.bmm(pp, vp).view(hkv, batch, q_len * GQA, d).transpose(0, 1)
    o = o + torch.bmm(ps.reshape(batch * hkv, q_len * GQA, most), vs).view(batch, hkv, q_len * GQA, d)
    o = o / torch.where(total == 0, torch.ones_like(total), total)[..., None]
    o = o.view(batch, hkv, q_len, GQA, d).transpose(1, 2)
    return o.reshape(q.shape).to(q.dtype)


def _plain_verify(st):
    target, draft, tokens, counts = st["target"], st["draft"], st["tokens"].long(), st["counts"].long()
    batch, k = tokens.shape
    b, i = torch.arange(batch, device=target.device), torch.arange(k, device=target.device)
    px = torch.gather(target[:, :k], 2, tokens[..., None])[..., 0].double()
    qx = torch.ones_like(px) if draft is None else torch.gather(draft, 2, tokens[..., None])[..., 0].double()
    taken = (st["accept_u"].double() * qx < px) & (i < counts[:, None])
    acc = taken.long().cumprod(1).sum(1)
    p = target[b, acc].double()
    at = acc.clamp(max=k - 1)
    if draft is None:
        left = p.scatter(1, tokens[b, at][:, None], 0.0)
    else:
        left = (p - draft[b, at].double()).clamp_min(0.0)
    left = torch.where((acc < counts)[:, None] & (left.sum(1, keepdim=True) > 0), left, p)
    c = left.cumsum(1)
    new = (c <= st["sample_u"].double()[:, None] * c[:, -1:]).sum(1)
    full = torch.nn.functional.pad(tokens, (0, 1))
    j = torch.arange(k + 1, device=target.device)
    out = torch.where(j < acc[:, None], full, torch.where(j == acc[:, None], new[:, None], torch.full_like(full, -1)))
    return out, acc.to(torch.int32), (st["lens"] + acc + 1).to(torch.int32)


# ----------------------------------------------------------------- 64-bit restatements
def _whole_rows(cache, slots):
    """float64 K and V rows of slots, one region at a time."""
    k, ks, v, vs, vz = (x.flatten(0, 1) if x.is_contiguous() else x for x in cache["regions"])
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


def _exact_load(case, cache):
    parts = [_whole_rows(cache, _row_slots(cache["table"][b], f, n, case["ppb"]))
             for b, (f, n) in enumerate(zip(_ints(case["firsts"]), _ints(case["counts"])))]
    return torch.cat([k for k, _ in parts]), torch.cat([v for _, v in parts])


def _exact_shared(case, cache, q):
    hkv, d, q_len, ppb = case["hkv"], case["head_dim"], case["q_len"], case["ppb"]
    prefix = case["prefix"] // PAGE * PAGE
    q = q.double()
    amax = q.abs().amax(-1)
    step = torch.where(amax == 0, torch.ones_like(amax), amax / 127.0)
    y = q * (1.0 / step)[..., None]
    q = torch.where(y >= 0, torch.floor(y + 0.5), torch.ceil(y - 0.5)) * step[..., None]
    out = torch.zeros_like(q)
    kp, vp = _whole_rows(cache, _row_slots(cache["prefix_table"], 0, prefix, ppb))
    kp, vp = kp.transpose(0, 1).contiguous(), vp.transpose(0, 1).contiguous()
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        kb, vb = _whole_rows(cache, _row_slots(cache["table"][b], prefix, max(0, n - prefix), ppb))
        for h in range(hkv):
            rows = q[b * q_len : (b + 1) * q_len, GQA * h : GQA * (h + 1)].reshape(-1, d)
            keys = torch.cat((kp[h], kb[:, h]))[:n]
            s = torch.mm(rows, keys.t()) / math.sqrt(d)
            end = n - q_len + 1 + torch.arange(q_len, device=q.device).repeat_interleave(GQA)
            s.masked_fill_(torch.arange(n, device=q.device)[None, :] >= end[:, None], -math.inf)
            p = torch.softmax(s, dim=1).nan_to_num_(0.0)  # a row that sees no key
            o = torch.mm(p, torch.cat((vp[h], vb[:, h]))[:n])
            out[b * q_len : (b + 1) * q_len, GQA * h : GQA * (h + 1)] = o.view(q_len, GQA, d)
    return out


def _exact_verify(case, st):
    k = case["drafts"]
    out = torch.full((case["batch"], k + 1), -1, dtype=torch.int64)
    accepted, lens = [], st["lens"].tolist()
    for b, n in enumerate(st["counts"].tolist()):
        p = st["target"][b].double()
        q = None if st["draft"] is None else st["draft"][b].double()
        a = 0
        while a < n:
            x = int(st["tokens"][b, a])
            qx = 1.0 if q is None else float(q[a, x])
            if not float(st["accept_u"][b, a]) * qx < float(p[a, x]):
                break
            out[b, a] = x
            a += 1
        w = p[a].clone()
        if a < n:
            if q is None:
                w[int(st["tokens"][b, a])] = 0.0
            else:
                w = torch.relu(w - q[a])
            if float(w.sum()) == 0.0:
                w = p[a].clone()
        c = torch.cumsum(w, 0)
        at = torch.searchsorted(c, c[-1] * float(st["sample_u"][b]), right=True)
        out[b, a] = int(at)
        accepted.append(a)
    dev = st["target"].device
    return (out.to(dev), torch.tensor(accepted, dtype=torch.int32, device=dev),
            torch.tensor([n + a + 1 for n, a in zip(lens, accepted)], dtype=torch.int32, device=dev))


# ------------------------------------------------------------------------------ inputs
def _named(name, case):
    return case if name is None else {"name": name, **case}


def _shared(name, hkv, head_dim, dtype, q_len, prefix, own_tokens, ppb=1, bound=False):
    """``own_tokens``: tokens of each sequence behind the prefix, the step's own included (0: a padding request)."""
    return _named(name, {"kind": "shared", "hkv": hkv, "head_dim": head_dim, "dtype": dtype, "q_len": q_len,
                         "prefix": prefix, "own_tokens": own_tokens, "ppb": ppb, "bound": bound})


def _load(name, hkv, head_dim, dtype, firsts, counts, ppb=1, bound=False):
    return _named(name, {"kind": "load", "hkv": hkv, "head_dim": head_dim, "dtype": dtype, "firsts": firsts,
                         "counts": counts, "ppb": ppb, "bound": bound})


def _verify(name, batch, k, vocab, dtype, drafts, filtered, bound=False):
    return _named(name, {"kind": "verify", "batch": batch, "drafts": k, "vocab": vocab, "dtype": dtype, "how": drafts,
                         "filtered": filtered, "bound": bound})


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def _text(values):
    return " ".join(str(int(x)) for x in values)


def _ints(text):
    return [int(x) for x in text.split()]


def _generator(seed, what):
    return torch.Generator(device="cuda" if torch.cuda.is_available() else "cpu").manual_seed(1000003 * seed + what)


def _lengths(case):
    """Cached tokens of each sequence (0: padding)."""
    if case["kind"] == "load":
        return [f + n for f, n in zip(_ints(case["firsts"]), _ints(case["counts"]))]
    return [case["prefix"] + n if n else 0 for n in _ints(case["own_tokens"])]


def _cache(case, seed):
    """A pool of region-major pages, its five views, and the block table.

    K rows are int8 codes of channels of uneven size (as rotary keys have) with
    a scale a row, V rows uint4 codes with a scale and a zero point a row, at
    random physical blocks; a shared prefix is the same blocks in every row."""
    hkv, d, ppb = case["hkv"], case["head_dim"], case["ppb"]
    gen = _generator(seed, 1)
    dev = gen.device
    lens = _lengths(case)
    need = [-(-n // (PAGE * ppb)) for n in lens]
    same = case["prefix"] // (PAGE * ppb) if case["kind"] == "shared" else 0  # whole shared blocks
    head = -(-case["prefix"] // (PAGE * ppb)) if case["kind"] == "shared" else 0
    pool = head + sum(max(0, n - same) for n in need)
    pool += pool // 10 + 2
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(1000003 * seed + 2)).to(torch.int32)
    table = torch.zeros((len(lens), max(1, *need)), dtype=torch.int32)
    at = head
    for b, n in enumerate(need):
        if n:
            table[b, : min(same, n)] = perm[: min(same, n)]
            fresh = max(0, n - same)
            table[b, same:n] = perm[at : at + fresh]
            at += fresh
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
    table = table.to(dev)
    live = next((b for b, n in enumerate(lens) if n), 0)
    return {"raw": raw, "regions": regions, "table": table, "prefix_table": table[live]}


def _queries(case, seed):
    """Views of a fused qkv projection's rows, as a model hands them over."""
    hkv, d = case["hkv"], case["head_dim"]
    n = case["q_len"] * len(_ints(case["own_tokens"]))
    gen = _generator(seed, 3)
    buf = (0.5 * torch.randn((n, (GQA + 2) * hkv * d), generator=gen, device=gen.device)).to(_DTYPES[case["dtype"]])
    return buf[:, : GQA * hkv * d].unflatten(1, (GQA * hkv, d))


def _drafted(case, seed):
    """A step's probabilities, drafts and random numbers.

    The draft model's logits are the target's with noise; ``filtered`` leaves
    the few hundred likeliest tokens of each target row, as top-k / top-p
    sampling does; ``greedy`` drafts are the draft model's likeliest tokens,
    given without probabilities; sequences hold between 0 and all drafts."""
    b, k, v, dt = case["batch"], case["drafts"], case["vocab"], _DTYPES[case["dtype"]]
    gen = _generator(seed, 4)
    dev = gen.device
    target = torch.empty((b, k + 1, v), dtype=dt, device=dev)
    draft = None if case["how"] == "greedy" else torch.empty((b, k, v), dtype=dt, device=dev)
    tokens = torch.empty((b, k), dtype=torch.int32, device=dev)
    for lo in range(0, b, 16):
        m = min(16, b - lo)
        logits = 2.5 * torch.randn((m, k + 1, v), generator=gen, device=dev)
        guess = torch.softmax(logits[:, :k] + 0.7 * torch.randn((m, k, v), generator=gen, device=dev), -1)
        if case["filtered"]:
            kth = logits.topk(min(200, v), dim=-1).values[..., -1:]
            logits.masked_fill_(logits < kth, -math.inf)
        target[lo : lo + m] = torch.softmax(logits, -1).to(dt)
        if draft is None:
            tokens[lo : lo + m] = guess.argmax(-1).to(torch.int32)
        else:
            noise = torch.empty_like(guess).exponential_(generator=gen)
            tokens[lo : lo + m] = (guess / noise).argmax(-1).to(torch.int32)
            draft[lo : lo + m] = guess.to(dt)
    counts = torch.full((b,), k, dtype=torch.int32, device=dev)
    short = torch.rand((b,), generator=gen, device=dev) < 0.2
    counts = torch.where(short, torch.randint(0, k + 1, (b,), generator=gen, device=dev, dtype=torch.int32), counts)
    return {
        "target": target, "draft": draft, "tokens": tokens, "counts": counts,
        "accept_u": torch.rand((b, k), generator=gen, device=dev),
        "sample_u": torch.rand((b,), generator=gen, device=dev),
        "lens": torch.randint(1, 100000, (b,), generator=gen, device=dev, dtype=torch.int32),
        "out_tokens": torch.empty((b, k + 1), dtype=torch.int64, device=dev),
        "accepted": torch.empty((b,), dtype=torch.int32, device=dev),
        "next_lens": torch.empty((b,), dtype=torch.int32, device=dev),
    }
