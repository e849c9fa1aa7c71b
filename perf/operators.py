"""Operator cases: the paged key-value cache with its attention, and the pick over penalised logits.

A program that decodes with this package runs, between its matrix products, three operators on
fp32 activations:

* ``append``: rotate the new tokens' queries and keys by their positions and store keys and values
  in the pages of a cache (f16, bf16, or 8-bit codes with a scale per position and head).
* ``attention``: 1..16 new tokens of each request over that cache, each token seeing the positions
  up to its own.
* ``logits``: repetition, presence and frequency penalties, biases and a grammar mask on the
  requests' logits, and the greedy pick.

Head layouts are those of the 9B-class layer of the benchmark (32 query and 8 key-value heads of
128) and of the 9B profile that packs are checked against (16 and 4 heads of 256, 64 of them
rotated), with generic ones around them; vocabularies are the benchmark's heads (151936 and 248320).

``own`` false: the plain form, elementary torch operations in 32 bits.  ``own`` true: the calls a
user makes (kq.kv.PagedAttention, kq.sampling.Picker).
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
NONE = -1e30          # a row whose values are all at or below this has no pick


# ---------------------------------------------------------------------------------------- cases

def _append(name, type, seqs, tokens, first, q_heads, kv_heads, dim, rot, page, interleaved):
    return {"name": name, "kind": "append", "type": type, "seqs": seqs, "tokens": tokens, "first": first,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "page": page,
            "interleaved": interleaved}


def _attention(name, type, seqs, tokens, longest, ragged, q_heads, kv_heads, dim, page):
    return {"name": name, "kind": "attention", "type": type, "seqs": seqs, "tokens": tokens, "longest": longest,
            "ragged": ragged, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page}


def _logits(name, rows, vocab, history, biases, masked, write):
    return {"name": name, "kind": "logits", "rows": rows, "vocab": vocab, "history": history, "biases": biases,
            "masked": masked, "write": write}


def listed():
    return [
        # One request's next token: the call of a single-user token loop.
        _append("append_1", "bf16", 1, 1, 700, 32, 8, 128, 128, 16, False),
        # A serving batch's next tokens, far enough apart that no two share a page.
        _append("append_64", "f16", 64, 1, 500, 16, 4, 256, 64, 16, False),
        # Prompt chunks of three requests into an 8-bit cache, pairs side by side.
        _append("append_prompt_i8", "i8", 3, 341, 5, 32, 8, 128, 128, 32, True),
        # A long prompt's chunk, bound by memory.
        _append("append_prompt_4096", "bf16", 2, 2048, 0, 32, 8, 128, 128, 16, False),
        # A single-user token over a short context: latency.
        _attention("attention_short", "bf16", 1, 1, 611, False, 32, 8, 128, 16),
        # The same user far into a long document: one request has to fill the card.
        _attention("attention_long", "bf16", 1, 1, 100001, False, 32, 8, 128, 16),
        # Verify of four drafted tokens for eight requests in the 9B profile's head layout.
        _attention("attention_verify_4", "f16", 8, 4, 5003, True, 16, 4, 256, 64),
        # A ragged serving batch.
        _attention("attention_batch", "bf16", 48, 1, 8191, True, 32, 8, 128, 16),
        # The same from an 8-bit cache, longer.
        _attention("attention_batch_i8", "i8", 32, 1, 16384, True, 32, 8, 128, 32),
        # One request's logits with penalties, constrained by a grammar; only the pick is wanted.
        _logits("logits_1", 1, 151936, 900, 8, True, False),
        # A chat batch with penalties and biases, logits kept for the log-probabilities.
        _logits("logits_32", 32, 151936, 2000, 100, False, True),
        # A large constrained batch on the larger vocabulary.
        _logits("logits_128", 128, 248320, 4000, 20, True, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """A head layout: 1..8 key-value heads, 1..8 query heads for each."""
    kv = rng.choice([1, 2, 4, 5, 8, 8])
    return kv * rng.choice([1, 2, 4, 4, 7, 8]), kv


def draw(rng):
    """One more case of the same ranges: batches of 1 to 64 requests, contexts to 100 thousand positions, head sizes
    in steps of 16 to 256, pages of 8 to 256 positions, vocabularies from 4 to 260 thousand."""
    kind = rng.choice(["append", "attention", "attention", "logits"])
    most = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
    type = rng.choice(sorted(DTYPE))
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
    page = 1 << rng.randint(3, 8)
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        case = _append("", type, seqs, 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048), _log_int(rng, 1, 1500) - 1,
                       q_heads, kv_heads, dim, rng.choice([dim, dim, 16, dim // 2 // 8 * 8]), page, rng.random() < 0.4)
        while work(case)["bytes"] > most:
            case["tokens"] = case["tokens"] * 3 // 4
    elif kind == "attention":
        case = _attention("", type, _log_int(rng, 1, 64), rng.choice([1, 1, 2, 4, 5, 8, 16]), _log_int(rng, 16, 100000),
                          rng.random() < 0.7, q_heads, kv_heads, dim, page)
        # no more bytes, and no larger float copies in the plain form, than the largest listed case
        wide = max(_padded(c) for c in listed() if c["kind"] == kind)
        while work(case)["bytes"] > most or _padded(case) > wide:
            case["longest"] = case["longest"] * 3 // 4
            if case["longest"] < 512 and case["seqs"] > 1:
                case["seqs"] = (case["seqs"] + 1) // 2
    else:
        case = _logits("", _log_int(rng, 1, 256), _log_int(rng, 4000, 260000), _log_int(rng, 1, 8000) - 1,
                       rng.choice([0, 5, 100, 300]), rng.random() < 0.5, rng.random() < 0.6)
        while work(case)["bytes"] > most:
            case["rows"] = case["rows"] * 3 // 4
    del case["name"]
    return case


def _lengths(case):
    """Context length of each request, new tokens included: all the longest, or spread evenly below it."""
    n, longest = case["seqs"], max(case["longest"], case["tokens"])
    if not case["ragged"]:
        return [longest] * n
    return [max(case["tokens"], longest * (i + 1) // n) for i in range(n)]


def _padded(case):
    """Keys of the plain form's float copy, in values."""
    return case["seqs"] * max(_lengths(case)) * case["kv_heads"] * case["dim"]


def _itemsize(case):
    return 1 if case["type"] == "i8" else 2


def work(case):
    if case["kind"] == "append":
        n, D = case["seqs"] * case["tokens"], case["dim"]
        scale = 4 if case["type"] == "i8" else 0
        per = 4 * D * (2 * case["q_heads"] + 2 * case["kv_heads"]) + 2 * case["kv_heads"] * (D * _itemsize(case) + scale)
        turned = (case["q_heads"] + case["kv_heads"]) * case["rot"]
        table = min(n, case["tokens"]) * case["rot"] * 4            # each position's cosines and sines once
        return {"bytes": n * (per + 8) + table, "flops": 3 * n * turned}
    if case["kind"] == "attention":
        total, T, D = sum(_lengths(case)), case["tokens"], case["dim"]
        scale = 4 if case["type"] == "i8" else 0
        cache = 2 * total * case["kv_heads"] * (D * _itemsize(case) + scale)
        rows = case["seqs"] * T * case["q_heads"]
        return {"bytes": cache + 8 * rows * D, "flops": 4 * total * T * case["q_heads"] * D}
    values = case["rows"] * case["vocab"]
    return {"bytes": values * (8 if case["write"] else 4) + (values // 8 if case["masked"] else 0)
            + case["rows"] * (4 * case["history"] + 8 * case["biases"] + 4), "flops": 2 * values}


# -------------------------------------------------------------------------------------- inputs

def _randn(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _pages(case, lengths, g):
    """A page table [seqs][width] whose pages lie anywhere in the pool, and the pool's size.  Entries past a request's
    pages are -1."""
    P, width = case["page"], -(-max(lengths) // case["page"])
    held = torch.tensor([-(-n // P) for n in lengths], device=DEV)
    used = torch.arange(width, device=DEV)[None] < held[:, None]
    pages = int(held.sum())
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
    table[used] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    return table, pages


def _rope_table(positions, rot):
    """[positions][rot] floats: the cosines of a position's angles, then the sines; angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "logits":
        return _prepare_logits(case, g, s)
    B, T, D, P = case["seqs"], case["tokens"], case["dim"], case["page"]
    Hq, Hkv, dt = case["q_heads"], case["kv_heads"], DTYPE[case["type"]]
    if case["kind"] == "append":
        # requests stand at different places of their contexts, each at or after `first`
        start = [case["first"] + 7 * i % 61 for i in range(B)]
        lengths = [n + T for n in start]
    else:
        lengths = _lengths(case)
        order = torch.randperm(B, generator=g, device=DEV).tolist()
        lengths = [lengths[i] for i in order]
    s["table"], pages = _pages(case, lengths, g)
    shape = (pages, Hkv, P, D)
    if case["kind"] == "append":
        s["k"], s["v"] = (torch.zeros(shape, dtype=dt, device=DEV) for _ in range(2))
        s["k_scale"], s["v_scale"] = ((torch.zeros(shape[:3], device=DEV) for _ in range(2)) if dt == torch.int8
                                      else (None, None))
        # q, k and v of a token as one projection writes them, side by side
        qkv = _randn((B * T, (Hq + 2 * Hkv) * D), g)
        s["q"], s["new_k"], s["new_v"] = qkv.split([Hq * D, Hkv * D, Hkv * D], 1)
        s["seq"] = torch.arange(B, device=DEV).repeat_interleave(T).to(torch.int32)
        s["pos"] = (torch.tensor(start, device=DEV)[:, None] + torch.arange(T, device=DEV)).reshape(-1).to(torch.int32)
        s["rope"] = _rope_table(s["table"].shape[1] * P, case["rot"])
        s["q_out"] = torch.empty((B * T, Hq * D), device=DEV)
        return s
    # keys with a few strong channels, as trained models have them
    channel = 1 + 3 * (torch.rand(D, generator=g, device=DEV) < 0.05)
    if dt == torch.int8:
        s["k"], s["v"] = (torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=dt) for _ in range(2))
        s["k_scale"], s["v_scale"] = ((1 + torch.rand(shape[:3], generator=g, device=DEV)) / 64 for _ in range(2))
    else:
        s["k"] = torch.empty(shape, dtype=dt, device=DEV).normal_(generator=g).mul_(channel.to(dt))
        s["v"] = torch.empty(shape, dtype=dt, device=DEV).normal_(generator=g)
        s["k_scale"] = s["v_scale"] = None
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    s["longest"] = max(lengths)
    s["q"] = _randn((B * T, Hq * D), g, 1.25)
    s["out"] = torch.empty((B * T, Hq * D), device=DEV)
    return s


def _prepare_logits(case, g, s):
    B, V, L, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    s["logits"] = _randn((B, V), g, 3.0)
    if L:
        # frequent tokens come again and again: ids spread over their logarithm
        u = torch.rand((B, L), generator=g, device=DEV)
        s["history"] = ((V ** u - 1).long() * 7919 % V).to(torch.int32)
        s["length"] = torch.randint(L // 2, L + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        s["prompt"] = s["length"] // 3
        s["repetition"] = 1 + torch.rand(B, generator=g, device=DEV) * 0.3
        s["frequency"], s["presence"] = (torch.rand(B, generator=g, device=DEV) * 0.6 for _ in range(2))
    if nb:
        step = V // nb                          # one id out of each stretch: all different
        s["bias_ids"] = (torch.arange(nb, device=DEV) * step
                         + torch.randint(0, step, (B, nb), generator=g, device=DEV)).to(torch.int32)
        s["bias_values"] = _randn((B, nb), g, 4.0)
    if case["masked"]:
        words = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, device=DEV)
        s["allowed"] = words.to(torch.int32)
    s["out"] = torch.empty((B, V), device=DEV) if case["write"] else None
    return s


# ---------------------------------------------------------------------------------- plain forms

def _turned(x, pos, rope, rot, interleaved):
    """x [N][heads][D] with the first rot values of each head rotated by its token's position."""
    cos, sin = rope[pos.long()][:, None].split(rot // 2, -1)
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _store(s, name, x, page, off):
    if s[name].dtype == torch.int8:
        scale = x.abs().amax(-1) / 127
        codes = torch.where(scale[..., None] > 0, x / scale[..., None], 0).round()
        s[name][page, :, off] = codes.to(torch.int8)
        s[name + "_scale"][page, :, off] = scale
    else:
        s[name][page, :, off] = x.to(s[name].dtype)


def _append_plain(s):
    case = s["case"]
    n, D, P, rot = s["q"].shape[0], case["dim"], case["page"], case["rot"]
    turn = (s["pos"], s["rope"], rot, case["interleaved"])
    page = s["table"][s["seq"].long(), (s["pos"] // P).long()].long()
    off = (s["pos"] % P).long()
    _store(s, "k", _turned(s["new_k"].reshape(n, -1, D), *turn), page, off)
    _store(s, "v", s["new_v"].reshape(n, -1, D), page, off)
    return _turned(s["q"].reshape(n, -1, D), *turn).reshape(n, -1)


def _stored(s, name):
    """The pool's values: 8-bit codes as the numbers they stand for."""
    return s[name] if s[name].dtype != torch.int8 else s[name] * s[name + "_scale"][..., None]


def _gathered(s, name):
    """[seqs][heads][positions][D] in 32 bits: every request's pages in order."""
    pages = s["table"].clamp(min=0).long()
    x = s[name][pages].float()
    if s[name].dtype == torch.int8:
        x = x * s[name + "_scale"][pages][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _attention_plain(s):
    case = s["case"]
    B, T, D, Hkv = case["seqs"], case["tokens"], case["dim"], case["kv_heads"]
    G = case["q_heads"] // Hkv
    k, v = _gathered(s, "k"), _gathered(s, "v")
    q = s["q"].view(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D)
    score = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    t = torch.arange(T, device=DEV).repeat_interleave(G)
    upto = s["lens"][:, None] - T + 1 + t                                   # positions that row t sees
    seen = torch.arange(k.shape[2], device=DEV) < upto[:, None, :, None]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total == 0, 1, total)
    return o.view(B, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B * T, -1)


def _logits_plain(s):
    y = s["logits"]
    B, V = y.shape
    if "history" in s:
        at = torch.arange(s["history"].shape[1], device=DEV)[None]
        ids, valid = s["history"].long(), at < s["length"][:, None]
        seen = torch.zeros_like(y).scatter_add_(1, ids, valid.float()) > 0
        count = torch.zeros_like(y).scatter_add_(1, ids, (valid & (at >= s["prompt"][:, None])).float())
        rep = s["repetition"][:, None]
        y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
        y = y - s["frequency"][:, None] * count
        y = y - s["presence"][:, None] * (count > 0)
    if "bias_ids" in s:
        y = y + torch.zeros_like(y).scatter_(1, s["bias_ids"].long(), s["bias_values"])
    if "allowed" in s:
        v = torch.arange(V, device=DEV)
        y = torch.where((s["allowed"][:, v >> 5] >> (v & 31)) & 1 != 0, y, -math.inf)
    top = y.amax(1, keepdim=True)
    picked = torch.where(y == top, torch.arange(V, device=DEV), V).amin(1)
    return y, torch.where(top[:, 0] > NONE, picked, -1).to(torch.int32)


# ------------------------------------------------------------------------------- the user's calls

def _handle(s):
    """What a serving program makes once: the attention over its cache with its workspace, or the picker."""
    path = os.path.join(ROOT, "oxcoder-9b_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kq import kv, sampling
    case = s["case"]
    if case["kind"] == "logits":
        return sampling.Picker(case["rows"], DEV)
    cache = kv.KVCache.over(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["kind"] == "append":
        return kv.PagedAttention([cache], s["table"], case["q_heads"], rope=s["rope"], interleaved=case["interleaved"])
    return kv.PagedAttention([cache], s["table"], case["q_heads"], tokens=case["tokens"], max_len=s["longest"])


def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        h = s.get("handle")
        if h is None:
            h = s["handle"] = _handle(s)
        if kind == "append":
            h.append(0, s["q"], s["new_k"], s["new_v"], s["seq"], s["pos"], s["q_out"])
            return {"q": s["q_out"], "k": _stored(s, "k"), "v": _stored(s, "v")}
        if kind == "attention":
            return {"out": h.attend(0, s["q"], s["lens"], s["out"])}
        picked = h.pick(s["logits"], history=s.get("history"), length=s.get("length"), prompt=s.get("prompt"),
                        repetition=s.get("repetition"), frequency=s.get("frequency"), presence=s.get("presence"),
                        bias_ids=s.get("bias_ids"), bias_values=s.get("bias_values"), allowed=s.get("allowed"),
                        out=s["out"])
        return {"picked": picked, "logits": s["out"]}
    if kind == "append":
        q = _append_plain(s)
        return {"q": q, "k": _stored(s, "k"), "v": _stored(s, "v")}
    if kind == "attention":
        return {"out": _attention_plain(s)}
    y, picked = _logits_plain(s)
    return {"picked": picked, "logits": y if s["out"] is not None else None}


# ------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    if case["kind"] == "logits" and not case["write"]:
        return None                             # an index alone
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["kind"]](s, case)


def _exact_append(s, case):
    """Rotation as a product of complex numbers; an 8-bit cache's codes have no value of their own in 64 bits."""
    n, D, rot = s["q"].shape[0], case["dim"], case["rot"]
    angle = torch.complex(*(x.double() for x in s["rope"][s["pos"].long()].chunk(2, 1)))[:, None]

    def turn(x):
        x = x.double().reshape(n, -1, D).clone()
        part = x[..., :rot]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(n, -1, rot // 2, 2).contiguous()) * angle
            x[..., :rot] = torch.view_as_real(z).reshape(n, -1, rot)
        else:
            z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * angle
            x[..., :rot // 2], x[..., rot // 2:rot] = z.real, z.imag
        return x

    q = turn(s["q"]).reshape(n, -1)
    if case["type"] == "i8":
        return {"q": q, "k": None, "v": None}
    out = {"q": q}
    place = s["pos"].long() // case["page"]
    for name, x in (("k", turn(s["new_k"])), ("v", s["new_v"].double().reshape(n, -1, D))):
        pool = torch.zeros(s[name].shape, dtype=torch.float64, device=DEV).transpose(1, 2)      # [page][position][head]
        pool[s["table"].long()[s["seq"].long(), place], s["pos"].long() - place * case["page"]] = x
        out[name] = pool.transpose(1, 2)
    return out


def _exact_attention(s, case):
    """Request by request and head by head, a softmax over the positions that a row sees."""
    T, D, P, Hq, Hkv = case["tokens"], case["dim"], case["page"], case["q_heads"], case["kv_heads"]
    out = torch.zeros((case["seqs"], T, Hq, D), dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, : -(-n // P)].long()
        for h in range(Hkv):
            kv = []
            for name in ("k", "v"):
                x = s[name][pages, h].double()
                if case["type"] == "i8":
                    x = x * s[name + "_scale"][pages, h].double()[..., None]
                kv.append(x.reshape(-1, D)[:n])
            mine = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            q = s["q"].view(case["seqs"], T, Hq, D)[b, :, mine].double()
            for t in range(T):
                m = n - T + 1 + t
                p = torch.softmax(q[t] @ kv[0][:m].T / math.sqrt(D), -1)
                out[b, t, mine] = p @ kv[1][:m]
    return {"out": out.reshape(case["seqs"] * T, -1)}


def _exact_logits(s, case):
    y = s["logits"].double()
    B, V = y.shape
    for b in range(B):
        row = y[b]
        if "history" in s:
            n, m = int(s["length"][b]), int(s["prompt"][b])
            ids = s["history"][b, :n].long()
            some = ids.unique()
            rep = s["repetition"][b].double()
            row[some] = torch.where(row[some] > 0, row[some] / rep, row[some] * rep)
            again, count = ids[m:].unique(return_counts=True)
            row[again] -= s["frequency"][b].double() * count + s["presence"][b].double()
        if "bias_ids" in s:
            row[s["bias_ids"][b].long()] += s["bias_values"][b].double()
        if "allowed" in s:
            bits = torch.stack([s["allowed"][b] >> i & 1 for i in range(32)], 1).reshape(-1)[:V]
            row[bits == 0] = -math.inf
    return {"picked": None, "logits": y}
