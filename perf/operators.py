"""Timed cases of the int8 key/value cache and of the attention over it.

A decoder that serves keeps the keys and values of its sequences as int8 codes in pages.  Three operations work on
them: rows of new tokens are quantized into their pages (`write`, read back here so that the values they stand for can be
seen), whole sequences come back as f32 (`read`), and new tokens attend over what their sequence has in the cache
(`attend`): one token of each sequence, a few drafted ones, a chunk of a prompt, a whole prompt, or queries over the
states of an encoder.

A page holds `page` tokens of every key/value head.  For each head it has, one after the other: codes of the keys
[dim / 16, page, 16], codes of the values [page / 16, dim, 16] (the last axis runs over tokens), the keys' scales
and the values' scales (f32, [page] each); head dimensions are rounded up to 16.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False


def listed():
    return [
        # One sequence, early on: the smallest call a program makes.
        {"name": "decode_1x300", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "rows": 1, "length": 300, "causal": True, "ragged": False},
        # A batch of sequences of all lengths, some of its places idle.
        {"name": "decode_48x6000", "op": "attend", "batch": 48, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "rows": 1, "length": 6000, "causal": True, "ragged": True},
        # Two long documents.
        {"name": "decode_2x65000", "op": "attend", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128,
         "rows": 1, "length": 65000, "causal": True, "ragged": False},
        # Five drafted tokens of each sequence, as many key/value heads as heads.
        {"name": "drafts_8x5", "op": "attend", "batch": 8, "heads": 16, "kv_heads": 16, "dim": 64, "page": 16,
         "rows": 5, "length": 3001, "causal": True, "ragged": True},
        # A prompt in chunks: a late chunk, and the odd last ones of several sequences (five heads a group, dim 80).
        {"name": "chunk_2048_of_16384", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "rows": 2048, "length": 16384, "causal": True, "ragged": False},
        {"name": "chunks_3x201_dim80", "op": "attend", "batch": 3, "heads": 20, "kv_heads": 4, "dim": 80, "page": 32,
         "rows": 201, "length": 1777, "causal": True, "ragged": True},
        # A prompt at once.
        {"name": "prompt_4096", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "rows": 4096, "length": 4096, "causal": True, "ragged": False},
        # Queries of a decoder over the states of an encoder, all of them visible.
        {"name": "encoder_states_4x1500", "op": "attend", "batch": 4, "heads": 12, "kv_heads": 12, "dim": 64, "page": 64,
         "rows": 77, "length": 1500, "causal": False, "ragged": False},
        # The new token of each sequence on its way into the cache; a prompt's.
        {"name": "write_64", "op": "write", "batch": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "rows": 1, "length": 900, "ragged": True},
        {"name": "write_prompts_2x8192", "op": "write", "batch": 2, "kv_heads": 8, "dim": 128, "page": 64,
         "rows": 8192, "length": 9000, "ragged": False},
        # Sequences back as f32, to go on with them elsewhere: all tokens of each, odd lengths.
        {"name": "read_6x5001", "op": "read", "batch": 6, "kv_heads": 8, "dim": 128, "page": 32,
         "rows": 5001, "length": 5001, "ragged": True},
        # One short sequence, a head dimension that is no multiple of 16.
        {"name": "read_1x333_dim72", "op": "read", "batch": 1, "kv_heads": 4, "dim": 72, "page": 16,
         "rows": 333, "length": 333, "ragged": False},
    ]


def _log_size(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "attend", "write", "read"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    dim = rng.choice([64, 64, 72, 80, 96, 128, 128, 128, 256])
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "ragged": rng.random() < 0.5}
    if op != "attend":
        case["batch"] = _log_size(rng, 1, 64)
        most = max(2, min(8192, (1 << 17) // case["batch"] // kv_heads))
        case["rows"] = _log_size(rng, 1, most)
        case["length"] = case["rows"] if op == "read" else case["rows"] + rng.randrange(0, 1000)
        return case
    kind = rng.choice(["decode", "decode", "drafts", "chunk", "chunk", "prompt", "states"])
    group = rng.choice([1, 2, 4, 4, 5, 8])
    case.update(heads=kv_heads * group, causal=kind != "states")
    if kind in ("decode", "drafts"):
        case["rows"] = 1 if kind == "decode" else rng.randrange(2, 9)
        case["batch"] = _log_size(rng, 1, 64)
        most = max(64, min(65536, (1 << 27) // (case["batch"] * kv_heads * dim)))
        case["length"] = max(case["rows"], _log_size(rng, 16, most))
    else:
        case["batch"] = rng.choice([1, 1, 2, 3, 4])
        case["rows"] = _log_size(rng, 16, 2048)
        # as many scores as the largest listed case has, and its work, at most
        most = min(16384, (1 << 29) // (case["rows"] * case["heads"] * case["batch"]))
        least = case["rows"] if case["causal"] else 16
        case["length"] = least if kind == "prompt" else max(least, _log_size(rng, 16, max(17, most)))
        while case["length"] * case["rows"] * case["heads"] * case["batch"] > 1 << 29:
            case["rows"] = (case["rows"] + 1) // 2
            case["length"] = max(case["rows"], case["length"] * 3 // 4) if kind != "prompt" else case["rows"]
    return case


def _sizes(case):
    """Each sequence's tokens in the cache, the new ones among them, and its rows in the call."""
    batch, rows, length = case["batch"], case["rows"], case["length"]
    lengths, counts = [], []
    for b in range(batch):
        part = (b * 0.6180339887) % 1.0 if case["ragged"] else 0.0
        n = rows - int(part * 0.7 * (rows - 1))
        at = length - int(part * 0.9 * length)
        if case["op"] == "read":
            at = n
        elif rows == 1 and case["ragged"] and case["op"] == "attend" and b % 8 == 7:
            at = 0                      # an idle place in the batch
        elif case.get("causal", True):
            at = max(at, n)
        lengths.append(at)
        counts.append(n)
    return lengths, counts


def _views(pages, case):
    """The keys' codes, the values' codes, and both scales, as they lie in the pages."""
    d, page = -(-case["dim"] // 16), case["page"]
    half = 16 * d * page
    codes, floats = pages.view(torch.int8), pages.view(torch.float32)
    return (codes[..., :half].unflatten(-1, (d, page, 16)), codes[..., half:2 * half].unflatten(-1, (page // 16, 16 * d, 16)),
            floats[..., half // 2:half // 2 + page], floats[..., half // 2 + page:])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    batch, kv_heads, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    lengths, counts = _sizes(case)
    wide = max(1, max(-(-n // page) for n in lengths))
    used = sum(-(-n // page) for n in lengths)
    num_pages = used + 3
    padded = 16 * -(-dim // 16)
    pages = torch.zeros(num_pages, kv_heads, page * (2 * padded + 8), dtype=torch.uint8, device="cuda")
    for codes in _views(pages, case)[:2]:
        codes.copy_((torch.randn(codes.shape, generator=gen, device="cuda") * 42.0).round_().clamp_(-127, 127))
    for scales in _views(pages, case)[2:]:
        scales.copy_((torch.rand(scales.shape, generator=gen, device="cuda") + 0.5) * (3.0 / 127.0))
    order = torch.randperm(num_pages, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.zeros(batch, wide, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lengths):
        n = -(-n // page)
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    s = {"case": dict(case), "pages": pages, "table": table, "num_pages": num_pages, "rows": starts[-1],
         "most_rows": max(counts), "most_length": max(lengths),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")}
    if case["op"] == "attend":
        s["q"] = torch.randn(starts[-1], case["heads"], dim, generator=gen, device="cuda") * 2.0
        s["scale"] = dim ** -0.5
    elif case["op"] == "write":
        # the projection that gives both: keys with a few large channels, one row in front of the other
        kv = torch.randn(starts[-1], 2 * kv_heads, dim, generator=gen, device="cuda")
        kv[:, :kv_heads, ::17] *= 6.0
        s["k"], s["v"] = kv[:, :kv_heads], kv[:, kv_heads:]
    return s


# -- the plain forms -----------------------------------------------------------------------

def _positions(s):
    """For each row of the call its sequence and its position there."""
    r = torch.arange(s["rows"], device="cuda")
    b = (r[:, None] >= s["starts"][None, 1:]).sum(1)
    return b, s["lengths"][b].long() - s["starts"][b + 1].long() + r


def _places(s):
    b, at = _positions(s)
    return s["table"][b, at // s["case"]["page"]].long(), at % s["case"]["page"]


def _quantize(x):
    # both quotients are 32-bit numbers by definition, correctly rounded: next to a border the last bit decides on the code
    scale = (x.abs().amax(-1).double() / 127.0).float()
    q = torch.round((x.double() / scale[..., None].double()).float()).clamp(-127, 127)
    return torch.where(scale[..., None] > 0, q, torch.zeros_like(q)).to(torch.int8), scale


def _gathered(s, page, slot):
    """Keys and values as f32, [..., kv_heads, dim], of the tokens at (page, slot)."""
    dim = s["case"]["dim"]
    kc, vc, ks, vs = _views(s["pages"], s["case"])
    k = kc[page, :, :, slot].flatten(-2)[..., :dim].float() * ks[page, :, slot][..., None]
    v = vc[page, :, slot // 16, :, slot % 16][..., :dim].float() * vs[page, :, slot][..., None]
    return k, v


def _plain_write(s):
    page, slot = _places(s)
    kc, vc, ks, vs = _views(s["pages"], s["case"])
    (k, sk), (v, sv) = _quantize(s["k"]), _quantize(s["v"])
    pad = 16 * -(-s["case"]["dim"] // 16) - s["case"]["dim"]
    k, v = torch.nn.functional.pad(k, (0, pad)), torch.nn.functional.pad(v, (0, pad))
    kc[page, :, :, slot] = k.unflatten(-1, (-1, 16))
    vc[page, :, slot // 16, :, slot % 16] = v
    ks[page, :, slot], vs[page, :, slot] = sk, sv


def _plain_read(s):
    return _gathered(s, *_places(s))


def _plain_attend(s):
    case = s["case"]
    heads, kv_heads, dim, batch = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    group, wide, most = heads // kv_heads, s["most_rows"], s["most_length"]
    j = torch.arange(most, device="cuda")
    k, v = _gathered(s, s["table"][:, j // case["page"]].long(), (j % case["page"]).expand(batch, most))
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    i = torch.arange(wide, device="cuda")
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    row = (s["starts"][:-1, None] + i).clamp(max=s["rows"] - 1).long()
    q = s["q"][row].unflatten(2, (kv_heads, group)).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * wide, dim)
    score = (torch.matmul(q, k) * s["scale"]).view(batch, kv_heads, group, wide, most)
    lengths = s["lengths"].long()
    last = lengths[:, None] - counts[:, None] + i if case["causal"] else (lengths[:, None] - 1).expand(batch, wide)
    seen = (j[None, None] <= last[:, :, None]) & (j[None, None] < lengths[:, None, None])
    seen = seen[:, None, None]
    score.masked_fill_(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(batch, kv_heads, group * wide, most), v).view(batch, kv_heads, group, wide, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(batch, wide, heads, dim)
    return out[i[None] < counts[:, None]]


# -- the framework's operators ---------------------------------------------------------------

def _handles(s):
    from vtl_amd import capi
    case = s["case"]
    cache = capi.KVCache(s["pages"].data_ptr(), s["num_pages"], case["page"], case["kv_heads"], case["dim"])
    starts = None if s["most_rows"] == 1 else s["starts"].data_ptr()    # one row each
    batch = capi.KVBatch(case["batch"], s["table"].shape[1], s["table"].data_ptr(), s["lengths"].data_ptr(), starts,
                         s["rows"], s["most_rows"], s["most_length"])
    return capi, ctypes.byref(cache), ctypes.byref(batch)


def _own_write(s):
    capi, cache, batch = _handles(s)
    k, v = s["k"], s["v"]
    capi.call("vtl_hip_kv_write_f32", cache, batch, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0))


def _own_read(s):
    capi, cache, batch = _handles(s)
    case = s["case"]
    k = torch.empty(s["rows"], case["kv_heads"], case["dim"], device="cuda")
    v = torch.empty_like(k)
    capi.call("vtl_hip_kv_read_f32", cache, batch, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0))
    return k, v


def _own_attend(s):
    capi, cache, batch = _handles(s)
    q, case = s["q"], s["case"]
    out = torch.empty_like(q)
    capi.call("vtl_hip_attention_i8_f32", cache, batch, q.data_ptr(), q.stride(0), case["heads"], s["scale"], int(case["causal"]),
              out.data_ptr(), out.stride(0), None, 0)
    return out


def run(s):
    op = s["case"]["op"]
    if op == "write":
        if own:
            _own_write(s)
            return _own_read(s)
        _plain_write(s)
        return _plain_read(s)
    if op == "read":
        return _own_read(s) if own else _plain_read(s)
    return _own_attend(s) if own else _plain_attend(s)


def work(case):
    lengths, counts = _sizes(case)
    kv_heads, dim = case["kv_heads"], case["dim"]
    token = kv_heads * (2 * dim + 8)             # a token in the cache: codes and scales
    if case["op"] != "attend":
        n = sum(counts)
        values = n * kv_heads * 2 * dim
        if case["op"] == "read":
            return {"bytes": n * token + 4 * values, "flops": values}
        return {"bytes": 4 * values + n * token + n * token + 4 * values, "flops": 4 * values}
    heads = case["heads"]
    pairs = seen = 0
    for at, n in zip(lengths, counts):
        first = at - n if case["causal"] else at - 1      # the last token that the first row sees
        step = 1 if case["causal"] else 0
        top = min(n, at) if case["causal"] else (n if at else 0)
        if top:
            low = max(first, 0) + 1
            pairs += top * low + step * top * (top - 1) // 2
            seen += at
    return {"bytes": seen * token + 8 * sum(counts) * heads * dim, "flops": 4 * dim * heads * pairs}


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    dim, kv_heads, page = case["dim"], case["kv_heads"], case["page"]
    lengths, counts = _sizes(case)
    padded = 16 * -(-dim // 16)
    half, block = padded * page, page * (2 * padded + 8)
    raw = s["pages"].reshape(-1)

    def tokens(b, first, n):
        """Keys and values of n tokens of sequence b from `first` on, [n, kv_heads, dim] in 64 bits."""
        at = torch.arange(first, first + n, device="cuda")
        base = (s["table"][b].long()[at // page][:, None] * kv_heads + torch.arange(kv_heads, device="cuda")) * block
        slot, d = at % page, torch.arange(dim, device="cuda")
        k_at = ((d // 16)[None] * page + slot[:, None]) * 16 + (d % 16)[None]
        v_at = half + ((slot // 16)[:, None] * padded + d[None]) * 16 + (slot % 16)[:, None]
        out = []
        for i, where in enumerate((k_at, v_at)):
            codes = raw.view(torch.int8)[base[:, :, None] + where[:, None]].double()
            scale = raw.view(torch.float32)[(base + 2 * half) // 4 + (slot + i * page)[:, None]]
            out.append(codes * scale.double()[..., None])
        return out

    if case["op"] == "write":
        back = []
        for x in (s["k"], s["v"]):
            # the scale is a 32-bit number by definition, and the code the nearest to the 32-bit quotient
            scale = (x.double().abs().amax(-1, keepdim=True) / 127.0).float()
            code = torch.round((x.double() / scale.double()).float().double()).clamp(-127, 127)
            back.append(torch.where(scale > 0, code * scale.double(), torch.zeros_like(code)))
        return tuple(back)
    if case["op"] == "read":
        parts = [tokens(b, lengths[b] - counts[b], counts[b]) for b in range(case["batch"])]
        return tuple(torch.cat([p[i] for p in parts]) for i in range(2))
    group = case["heads"] // kv_heads
    out = torch.zeros(s["rows"], case["heads"], dim, dtype=torch.float64, device="cuda")
    row = 0
    for b in range(case["batch"]):
        n, at = counts[b], lengths[b]
        if at:
            keys, values = tokens(b, 0, at)
            for lo in range(kv_heads):
                k, v = keys[:, lo].contiguous(), values[:, lo].contiguous()
                q = s["q"][row:row + n, lo * group:(lo + 1) * group].double()
                score = torch.matmul(q.reshape(n * group, dim), k.T.contiguous()).view(n, group, at) * s["scale"]
                if case["causal"]:
                    last = torch.arange(n, device="cuda") + at - n
                    score.masked_fill_((torch.arange(at, device="cuda")[None] > last[:, None])[:, None], float("-inf"))
                weight = torch.softmax(score, -1)
                out[row:row + n, lo * group:(lo + 1) * group] = torch.matmul(weight.view(n * group, at), v).view(n, group, dim)
        row += n
    return out
