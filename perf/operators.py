"""Cases, inputs and plain forms of the operators that take a prompt into the paged cache and attend to it.

Three operators, each measured as a user's program calls it:

* ``append``  ``rope_append_kv``: rotary positions on q and k, K and V rows into their pages, the INT4
  slabs and the page metadata that the decode step reads, for any number of new tokens per sequence; the
  cases with INT4 slabs also read the written pages back (``dequantize_k_pages``).
* ``prefix``  ``shared_prefix_attn``: decode attention of groups of sequences over a prefix that a group
  shares, read once per group, and over each sequence's own pages.
* ``prompt``  ``prompt_attn``: causal attention of a ragged batch's new tokens over the paged cache; with a
  token budget, over the pages that ``quest_select_blocks`` picks for every block of queries.

``run`` computes them in elementary torch operations in 32 bits (angles in 64), or, with ``own`` set, calls
the operators.  ``exact`` computes the same in 64 bits, sequence by sequence.
"""
import math
import random

import torch

own = False

PAGE, D, GROUP = 16, 128, 32
SM_SCALE = 1.0 / math.sqrt(D)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one token each for a small batch: a decode step's append, all latency (8 KV heads, 32 query heads)
        {"name": "append decode b8", "op": "append", "batch": 8, "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 2000, "hq": 32, "hkv": 8,
         "dtype": "bf16", "rotary": 128, "inter": False, "scaling": "none", "far": 0, "k4": True, "lengths": 1},
        # a large decode batch without grouped heads, interleaved pairs on half of the head
        {"name": "append decode b256 mha", "op": "append", "batch": 256, "new_lo": 1, "new_hi": 1, "old_lo": 0, "old_hi": 300, "hq": 32,
         "hkv": 32, "dtype": "fp16", "rotary": 64, "inter": True, "scaling": "none", "far": 0, "k4": True,
         "lengths": 2},
        # ragged prompts entering an empty cache
        {"name": "append prompts ragged", "op": "append", "batch": 6, "new_lo": 60, "new_hi": 8192, "old_lo": 0, "old_hi": 0, "hq": 32,
         "hkv": 8, "dtype": "bf16", "rotary": 128, "inter": False, "scaling": "llama3", "far": 0, "k4": True,
         "lengths": 3},
        # chunks of long contexts: far positions, frequencies scaled for them, no INT4 slabs
        {"name": "append chunks far", "op": "append", "batch": 4, "new_lo": 500, "new_hi": 4096, "old_lo": 1, "old_hi": 100, "hq": 64,
         "hkv": 8, "dtype": "bf16", "rotary": 128, "inter": False, "scaling": "yarn", "far": 120000, "k4": False,
         "lengths": 4},
        # four sequences over one short system prompt
        {"name": "prefix short b4", "op": "prefix", "batch": 4, "groups": 1, "prefix_lo": 300, "prefix_hi": 300, "own_lo": 0, "own_hi": 40,
         "hq": 32, "hkv": 8, "dtype": "bf16", "lengths": 5},
        # the decode batch of 64 over one 32K document
        {"name": "prefix 32k b64", "op": "prefix", "batch": 64, "groups": 1, "prefix_lo": 32768, "prefix_hi": 32768,
         "own_lo": 1, "own_hi": 512, "hq": 32, "hkv": 8, "dtype": "bf16", "lengths": 6},
        # several documents, each asked about by some sequences; every query head has its KV head
        {"name": "prefix groups fp16 mha", "op": "prefix", "batch": 96, "groups": 4, "prefix_lo": 1000, "prefix_hi": 8000,
         "own_lo": 0, "own_hi": 300, "hq": 32, "hkv": 32, "dtype": "fp16", "lengths": 7},
        # many samples of one prompt: the shared part is a dense product
        {"name": "prefix 8k b256 g8", "op": "prefix", "batch": 256, "groups": 1, "prefix_lo": 8191, "prefix_hi": 8191,
         "own_lo": 1, "own_hi": 700, "hq": 64, "hkv": 8, "dtype": "bf16", "lengths": 8},
        # a few tokens each behind short contexts
        {"name": "prompt small", "op": "prompt", "batch": 3, "new_lo": 1, "new_hi": 40, "old_lo": 0, "old_hi": 700, "hq": 32, "hkv": 8,
         "dtype": "bf16", "budget": 0, "block": 64, "lengths": 9},
        # ragged prompts, dense (the layers that are not sparsified)
        {"name": "prompt ragged dense", "op": "prompt", "batch": 4, "new_lo": 700, "new_hi": 4096, "old_lo": 0, "old_hi": 1000, "hq": 32,
         "hkv": 8, "dtype": "bf16", "budget": 0, "block": 64, "lengths": 10},
        # a chunk of a 32K prompt, every block of 64 queries over its 4096 best tokens
        {"name": "prompt chunk 32k sparse", "op": "prompt", "batch": 1, "new_lo": 4096, "new_hi": 4096, "old_lo": 28672, "old_hi": 28672,
         "hq": 32, "hkv": 8, "dtype": "bf16", "budget": 4096, "block": 64, "lengths": 11},
        # two prompts without grouped heads, sparse
        {"name": "prompt sparse fp16 mha", "op": "prompt", "batch": 2, "new_lo": 2000, "new_hi": 4096, "old_lo": 0, "old_hi": 4096,
         "hq": 16, "hkv": 16, "dtype": "fp16", "budget": 1024, "block": 128, "lengths": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: batches, lengths, head groupings, types and layouts."""
    op = rng.choice(["append", "prefix", "prompt"])
    hq, hkv = rng.choice([(32, 8), (32, 32), (64, 8), (32, 4), (28, 4), (16, 16), (24, 8), (8, 1), (40, 8)])
    c = {"op": op, "hq": hq, "hkv": hkv, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "lengths": rng.randrange(1 << 20)}
    if op == "append":
        batch = _log(rng, 1, 256)
        most = max(1, 16000 * 40 // (hq + 2 * hkv) // batch)
        hi = _log(rng, 1, min(8192, most))
        c.update(batch=batch, new_lo=max(1, hi // rng.choice([1, 2, 30])), new_hi=hi, old_lo=0, old_hi=_log(rng, 1, 400),
                 rotary=rng.choice([128, 128, 64, 32, 96]), inter=rng.random() < 0.4,
                 scaling=rng.choice(["none", "linear", "llama3", "yarn"]), far=rng.choice([0, 0, _log(rng, 100, 200000)]),
                 k4=rng.random() < 0.6)
    elif op == "prefix":
        batch = _log(rng, 1, 256)
        groups = min(batch, rng.choice([1, 1, 2, 5]))
        p = _log(rng, 16, min(32768, 2_000_000 // (batch * max(1, hq // 32))))
        hi = _log(rng, 1, max(2, min(2048, 64 * 512 // batch)))
        c.update(batch=batch, groups=groups, prefix_lo=max(1, p // rng.choice([1, 3])), prefix_hi=p,
                 own_lo=rng.choice([0, 1]), own_hi=hi)
    else:
        batch = _log(rng, 1, 32)
        hi = _log(rng, 1, 4096 // batch + 1)
        old = _log(rng, 1, min(28672, 4096 * 32768 // (batch * hi * max(1, hq // 32))))
        sparse = rng.random() < 0.6
        c.update(batch=batch, new_lo=max(1, hi // rng.choice([1, 4, 20])), new_hi=hi, old_lo=rng.choice([0, old]), old_hi=old,
                 budget=_log(rng, 64, 4096) if sparse else 0, block=rng.choice([64, 64, 32, 128]))
    return c


def _lengths(case):
    """The whole numbers of a case, from the case alone: new/old tokens, or prefix/own tokens and group sizes."""
    rng = random.Random(case["lengths"])
    pick = lambda r: case[r + "_lo"] + int(round(rng.random() * (case[r + "_hi"] - case[r + "_lo"])))  # noqa: E731
    n = case["batch"]
    if case["op"] == "prefix":
        cuts = sorted(rng.sample(range(1, n), case["groups"] - 1)) if case["groups"] > 1 else []
        return {"prefix": [pick("prefix") for _ in range(case["groups"])],
                "own": [pick("own") for _ in range(n)], "group": [0] + cuts + [n]}
    return {"new": [pick("new") for _ in range(n)], "old": [pick("old") for _ in range(n)]}


def _selected(case, lens):
    """(tokens of K read per KV head summed over blocks, q.k pairs per query head) of a prompt case."""
    read = pairs = 0
    for n, o in zip(lens["new"], lens["old"]):
        if not case["budget"]:
            read += n + o
            pairs += n * o + n * (n + 1) // 2
            continue
        k = max(1, case["budget"] // PAGE) + (case["budget"] % PAGE != 0)
        for t in range(0, n, case["block"]):
            m = min(case["block"], n - t)
            history = min(k, (o + t) // PAGE) * PAGE
            inside = (o + t) % PAGE
            read += history + inside + m
            pairs += m * (history + inside) + m * (m + 1) // 2
    return read, pairs


def work(case):
    """Bytes and operations of one pass: every input that is needed read once, every output written once."""
    lens, hq, hkv = _lengths(case), case["hq"], case["hkv"]
    if case["op"] == "append":
        t = sum(lens["new"])
        b = t * (hq + 2 * hkv) * D * 2 * 2                     # q, k, v in; q and the K and V rows out
        pages = sum((n + o + PAGE - 1) // PAGE - o // PAGE for n, o in zip(lens["new"], lens["old"]))
        b += pages * hkv * 2 * D * 2                           # page metadata out
        if case["k4"]:
            b += t * hkv * 80                                  # INT4 slabs out
            b += pages * hkv * (1280 + PAGE * D * 2)           # and read back
        return {"bytes": b, "flops": t * (hq + hkv) * case["rotary"] * 3}
    if case["op"] == "prefix":
        n = case["batch"]
        shared, mine = sum(lens["prefix"]), sum(lens["own"])
        size = [lens["group"][i + 1] - lens["group"][i] for i in range(case["groups"])]
        pairs = sum(s * p for s, p in zip(size, lens["prefix"])) + mine
        return {"bytes": (shared + mine) * hkv * D * 4 + 2 * n * hq * D * 2, "flops": 4 * pairs * hq * D}
    t = sum(lens["new"])
    read, pairs = _selected(case, lens)
    total = sum(lens["new"]) + sum(lens["old"])
    b = min(read, total) * hkv * D * 4 + 2 * t * hq * D * 2    # a token that several blocks keep counts once
    f = 4 * pairs * hq * D
    if case["budget"]:
        b += total // PAGE * hkv * 2 * D * 2
        f += sum(2 * 2 * D * hkv * ((o + s) // PAGE) for n, o in zip(lens["new"], lens["old"])
                 for s in range(0, n, case["block"]))
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _table(lens, first, order):
    """CSR page table of sequences of `lens` tokens (none for an empty one) on the physical pages `order[first:]`."""
    n = [(x + PAGE - 1) // PAGE for x in lens]
    ptr = [0]
    for x in n:
        ptr.append(ptr[-1] + x)
    last = _i32([(x - 1) % PAGE + 1 if x else 0 for x in lens])
    return _i32(ptr), order[first: first + ptr[-1]].to(torch.int32).contiguous(), last, ptr[-1]


def _pool(pages, hkv, dt, g):
    """K and V pages.  Keys lean towards a direction of their KV head, a few of them strongly, so that attention
    over them is neither flat nor one token's."""
    lean = torch.randn(hkv, 1, D, generator=g, device=DEV)
    k, v = (torch.empty(pages, hkv, PAGE, D, dtype=dt, device=DEV) for _ in range(2))
    step = max(1, (1 << 26) // (hkv * PAGE * D))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        heavy = torch.rand(b - a, hkv, PAGE, 1, generator=g, device=DEV) < 0.02
        k[a:b] = (torch.randn(b - a, hkv, PAGE, D, generator=g, device=DEV) + (0.1 + 0.5 * heavy) * lean).to(dt)
        v[a:b] = (torch.randn(b - a, hkv, PAGE, D, generator=g, device=DEV) + 0.2).to(dt)
    return k, v, lean


def _scaling(case):
    """Frequency scaling as a model's configuration states it."""
    return {"none": None, "linear": {"rope_type": "linear", "factor": 4.0},
            "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position_embeddings": 8192},
            "yarn": {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 8192}}[case["scaling"]]


BASE = 500000.0


def _frequencies(rotary, scaling):
    """Angle per position of every pair, in 64 bits, and the factor on cos and sin."""
    f = BASE ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    kind = scaling["rope_type"] if scaling else "none"
    if kind == "none":
        return f, 1.0
    s = scaling["factor"]
    if kind == "linear":
        return f / s, 1.0
    n = scaling["original_max_position_embeddings"]
    if kind == "llama3":
        lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
        turns = n * f / (2 * math.pi)
        mix = ((turns - lo) / (hi - lo)).clamp(0, 1)
        return f / s * (1 - mix) + f * mix, 1.0
    at = lambda turns: rotary * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rotary - 1)
    ramp = ((torch.arange(rotary // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f / s * ramp + f * (1 - ramp), 0.1 * math.log(s) + 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, hq, hkv, lens = DTYPES[case["dtype"]], case["hq"], case["hkv"], _lengths(case)
    s = {"case": case, "lens": lens}
    if case["op"] == "prefix":
        own_pages = sum((n + PAGE - 1) // PAGE for n in lens["own"])
        pages = own_pages + sum((n + PAGE - 1) // PAGE for n in lens["prefix"])
        order = torch.randperm(pages, generator=g, device=DEV)
        s["indptr"], s["indices"], s["last"], used = _table(lens["own"], 0, order)
        s["p_indptr"], s["p_indices"], s["p_last"], _ = _table(lens["prefix"], used, order)
        s["group"] = _i32(lens["group"])
        s["k"], s["v"], lean = _pool(pages, hkv, dt, g)
        s["q"] = _queries(case["batch"], hq, hkv, lean, dt, g)
        s["rows"] = torch.repeat_interleave(torch.arange(case["groups"], device=DEV),
                                            (s["group"][1:] - s["group"][:-1]).long())
        return s
    total = [n + o for n, o in zip(lens["new"], lens["old"])]
    pages = sum((n + PAGE - 1) // PAGE for n in total)
    order = torch.randperm(pages, generator=g, device=DEV)
    s["indptr"], s["indices"], s["last"], _ = _table(total, 0, order)
    ptr = [0]
    for n in lens["new"]:
        ptr.append(ptr[-1] + n)
    s["qo"] = _i32(ptr)
    s["k"], s["v"], lean = _pool(pages, hkv, dt, g)
    if case["op"] == "prompt":
        s["q"] = _queries(ptr[-1], hq, hkv, lean, dt, g)
        s["max_pages"] = max((n + PAGE - 1) // PAGE for n in total)
        s["meta"] = torch.stack([s["k"].amin(2), s["k"].amax(2)], 2).contiguous()
        for b, n in enumerate(total):  # the unused rows of a last page count for nothing
            if n % PAGE:
                page = int(s["indices"][int(s["indptr"][b + 1]) - 1])
                rows = s["k"][page, :, : n % PAGE]
                s["meta"][page, :, 0], s["meta"][page, :, 1] = rows.amin(1), rows.amax(1)
        return s
    # append: q, k and v are parts of one projection's output, as a model has them
    proj = torch.randn(ptr[-1], hq + 2 * hkv, D, generator=g, device=DEV).to(dt)
    s["new_q"], s["new_k"], s["new_v"] = proj[:, :hq], proj[:, hq: hq + hkv], proj[:, hq + hkv:]
    s["k4"] = _slabs(s["k"]) if case["k4"] else None
    s["meta"] = torch.stack([s["k"].amin(2), s["k"].amax(2)], 2).contiguous()
    freqs, s["factor"] = _frequencies(case["rotary"], _scaling(case))
    s["freqs"] = freqs.to(DEV)
    seq = torch.repeat_interleave(torch.arange(case["batch"], device=DEV), _i32(lens["new"]).long())
    s["slot"] = torch.arange(ptr[-1], device=DEV) - s["qo"].long()[seq] + _i32(lens["old"]).long()[seq]
    s["positions"] = s["slot"] + case["far"] if case["far"] else None
    s["page_of"] = s["indices"].long()[s["indptr"].long()[seq] + s["slot"] // PAGE]
    s["touched"] = torch.unique(s["page_of"])                   # the pages that get new tokens
    s["ids"] = s["touched"].to(torch.int32)
    return s


def _queries(rows, hq, hkv, lean, dt, g):
    q = torch.randn(rows, hkv, hq // hkv, D, generator=g, device=DEV) + 0.3 * lean[None]
    return q.reshape(rows, hq, D).to(dt)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"append": _append, "prefix": _prefix, "prompt": _prompt}[s["case"]["op"]](s)


def _append(s):
    c = s["case"]
    if own:
        from twilight_b200.kernel import ops
        q = ops.rope_append_kv(s["new_q"], s["new_k"], s["new_v"], s["freqs"], s["k"], s["v"], s["k4"], s["meta"],
                               s["qo"], s["indptr"], s["indices"], s["last"], positions=s["positions"],
                               interleaved=c["inter"], attention_scale=s["factor"])
        k4 = ops.dequantize_k_pages(s["k4"], s["ids"], dtype=q.dtype) if c["k4"] else None
    else:
        pos = s["slot"] if s["positions"] is None else s["positions"]
        angle = pos.double()[:, None] * s["freqs"]
        cos, sin = ((x * s["factor"]).float()[:, None] for x in (angle.cos(), angle.sin()))
        q, k = (_rotate(s[n].float(), cos, sin, c["rotary"], c["inter"]).to(s["k"].dtype) for n in ("new_q", "new_k"))
        s["k"][s["page_of"], :, s["slot"] % PAGE] = k
        s["v"][s["page_of"], :, s["slot"] % PAGE] = s["new_v"]
        _fold_meta(s, k)
        k4 = _quantised(s["k"][s["touched"]]) if c["k4"] else None
    out = {"q": q, "k": s["k"], "v": s["v"], "meta": s["meta"]}
    return {**out, "k4": k4} if c["k4"] else out


def _rotate(x, cos, sin, rotary, inter):
    r, rest = x[..., :rotary], x[..., rotary:]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., : rotary // 2], r[..., rotary // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([r, rest], -1)


def _fold_meta(s, k):
    """Channel-wise minimum and maximum of every page that got tokens: of its new rows, and of what it held before
    where its first row is an old one."""
    page, hkv = s["page_of"], k.shape[1]
    at = page[:, None, None].expand(-1, hkv, D)
    fresh = torch.zeros(s["k"].shape[0], dtype=torch.bool, device=DEV)
    fresh[page[s["slot"] % PAGE == 0]] = True
    for i, how, start in ((0, "amin", math.inf), (1, "amax", -math.inf)):
        was = torch.where(fresh[:, None, None], torch.full_like(s["meta"][:, :, i], start), s["meta"][:, :, i])
        s["meta"][:, :, i] = was.scatter_reduce(0, at, k, how)


def _codes(k):
    """4-bit codes per token and 32 channels, between the group's minimum and maximum, every step in the cache's type as
    the framework's quantiser defines it; a group without a range gets code 0 and scale 0."""
    x = k.unflatten(-1, (D // GROUP, GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = (hi - lo).clamp(min=1e-9) / 15
    code = ((x - lo) / scale).round().clamp(0, 15)
    return torch.where(scale > 0, code, torch.zeros_like(code)), scale, lo


def _quantised(k):
    """The values that the codes of `k` stand for."""
    code, scale, lo = _codes(k)
    return (code.float() * scale.half().float() + lo.half().float()).flatten(-2).to(k.dtype)


def _slabs(k):
    """INT4 slabs of whole pages: 16 x 64 code bytes (an even channel in the low nibble), then 16 x 4 x {scale, min}
    in fp16."""
    code, scale, lo = _codes(k)
    code = code.flatten(-2).to(torch.uint8).flatten(2)
    pairs = torch.cat([scale, lo], -1).half().flatten(2).contiguous().view(torch.uint8)
    return torch.cat([code[..., 0::2] | (code[..., 1::2] << 4), pairs], -1).contiguous()


def _gather(pool, ptr, indices, most):
    """[sequences, hkv, most*16, D] in 32 bits through the page table, and its token positions."""
    n = ptr[1:] - ptr[:-1]
    at = torch.arange(most, device=DEV)
    ids = torch.where(at < n[:, None], indices[(ptr[:-1, None] + at).clamp(max=max(0, indices.numel() - 1))], 0)
    return pool[ids.long()].permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _tokens(ptr, last):
    n = (ptr[1:] - ptr[:-1]).long()
    return torch.where(n > 0, (n - 1) * PAGE + last.long(), 0)


def _attend(q, k, v, keep):
    """softmax of q.k over the kept keys, times v; zeros where no key is kept.  Returns what two of them are joined by:
    maximum, sum, and the sum of the weighted values."""
    x = torch.matmul(q, k.transpose(-1, -2)) * SM_SCALE
    x = x.masked_fill(~keep, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _prefix(s):
    c, lens = s["case"], s["lens"]
    if own:
        from twilight_b200.kernel import ops
        return ops.shared_prefix_attn(s["q"], s["k"], s["v"], s["group"], s["p_indptr"], s["p_indices"], s["p_last"],
                                      s["indptr"], s["indices"], s["last"])
    n, hq, hkv, groups = c["batch"], c["hq"], c["hkv"], c["groups"]
    q = s["q"].float().unflatten(1, (hkv, hq // hkv))                                # [n, hkv, g, D]
    # the shared part: the sequences of a group are the rows of one product
    most = max((x + PAGE - 1) // PAGE for x in lens["prefix"])
    size = max(b - a for a, b in zip(lens["group"], lens["group"][1:]))
    k, v = (_gather(s[x], s["p_indptr"], s["p_indices"], most) for x in "kv")
    at = torch.arange(n, device=DEV) - s["group"].long()[s["rows"]]
    packed = torch.zeros(groups, hkv, size, hq // hkv, D, device=DEV)
    packed[s["rows"], :, at] = q
    keep = torch.arange(most * PAGE, device=DEV) < _tokens(s["p_indptr"], s["p_last"])[:, None, None, None]
    m, l, o = (x.unflatten(2, (size, hq // hkv))[s["rows"], :, at] for x in _attend(packed.flatten(2, 3), k, v, keep))
    # each sequence's own part
    most = max((x + PAGE - 1) // PAGE for x in lens["own"])
    if most:
        k, v = (_gather(s[x], s["indptr"], s["indices"], most) for x in "kv")
        keep = torch.arange(most * PAGE, device=DEV) < _tokens(s["indptr"], s["last"])[:, None, None, None]
        m2, l2, o2 = _attend(q, k, v, keep)
        top = torch.maximum(m, m2)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        a, b = torch.exp(m - top), torch.exp(m2 - top)
        l, o = l * a + l2 * b, o * a + o2 * b
    return (o / torch.where(l > 0, l, torch.ones_like(l))).flatten(1, 2).to(s["q"].dtype)


def _prompt(s):
    c, lens = s["case"], s["lens"]
    if own:
        from twilight_b200.kernel import ops
        pages = (None, None)
        if c["budget"]:
            pages = ops.quest_select_blocks(s["q"], s["meta"], s["qo"], s["indptr"], s["indices"], s["last"],
                                            c["budget"], max_pages=s["max_pages"], query_block=c["block"])
        return ops.prompt_attn(s["q"], s["k"], s["v"], s["qo"], s["indptr"], s["indices"], s["last"],
                               max_pages=s["max_pages"], block_pages=pages[0], block_npages=pages[1],
                               query_block=c["block"])
    n, hq, hkv, g = c["batch"], c["hq"], c["hkv"], c["hq"] // c["hkv"]
    most, size = s["max_pages"], -(-max(lens["new"]) // c["block"]) * c["block"]
    ptr, total = s["qo"].long(), _tokens(s["indptr"], s["last"])
    new = ptr[1:] - ptr[:-1]
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), new)
    at = torch.arange(seq.shape[0], device=DEV) - ptr[seq]
    q = torch.zeros(n, size, hq, D, device=DEV)                                      # padded, and zero there
    q[seq, at] = s["q"].float()
    where = (total - new)[:, None] + torch.arange(size, device=DEV)                  # positions of the queries
    keep = torch.arange(most * PAGE, device=DEV) <= where[..., None]                 # [n, size, tokens]
    keep &= torch.arange(most * PAGE, device=DEV) < total[:, None, None]
    keep = keep[:, None]
    if c["budget"]:
        keep = keep & _chosen(s, q, where, total, most).repeat_interleave(PAGE, -1)
    k, v = (_gather(s[x], s["indptr"], s["indices"], most) for x in "kv")
    rows = q.unflatten(2, (hkv, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)             # [n, hkv, g*size, D]
    keep = keep.expand(n, hkv, size, most * PAGE)[:, :, None].expand(n, hkv, g, size, most * PAGE).flatten(2, 3)
    m, l, o = _attend(rows, k, v, keep)
    o = (o / torch.where(l > 0, l, torch.ones_like(l))).unflatten(2, (g, size)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[seq, at].to(s["q"].dtype)


def _chosen(s, q, where, total, most):
    """[n, hkv, size, most] pages of every query: its block's own ones and, of those before the block, the budget's best
    by the block's summed bounds sum_d max(q_d*kmax_d, q_d*kmin_d); ties to the lower page."""
    c = s["case"]
    n, size, hq, _ = q.shape
    hkv, block = c["hkv"], c["block"]
    parts = q.unflatten(2, (hkv, hq // hkv)).unflatten(1, (size // block, block))
    lo, hi = parts.clamp(max=0).sum((2, 4)), parts.clamp(min=0).sum((2, 4))          # [n, blocks, hkv, D]
    ptr = s["indptr"]
    at = torch.arange(most, device=DEV)
    entry = (ptr[:-1, None] + at).clamp(max=s["indices"].numel() - 1)
    ids = torch.where(at < (ptr[1:] - ptr[:-1])[:, None], s["indices"][entry], 0)
    meta = s["meta"][ids.long()].float().permute(0, 2, 3, 4, 1)                      # [n, hkv, 2, D, pages]
    score = torch.matmul(lo.transpose(1, 2), meta[:, :, 0]) + torch.matmul(hi.transpose(1, 2), meta[:, :, 1])
    first = where[:, ::block]                                                        # [n, blocks]
    score = score.masked_fill((at >= (first // PAGE)[..., None])[:, None], -math.inf)
    k = max(1, c["budget"] // PAGE) + (c["budget"] % PAGE != 0)
    best = score.sort(stable=True, dim=-1, descending=True).indices[..., :k]
    chosen = torch.zeros_like(score, dtype=torch.bool).scatter(-1, best, True) & (score > -math.inf)
    chosen |= (at >= (first // PAGE)[..., None])[:, None]                            # the rest is cut by the causal mask
    return chosen.repeat_interleave(block, 2)


# ---------------------------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append64, "prefix": _prefix64, "prompt": _prompt64}[case["op"]](s)


def _append64(s):
    c, lens = s["case"], s["lens"]
    half = c["rotary"] // 2
    new = {"q": [], "k": []}
    cache_k, cache_v, meta = s["k"].double(), s["v"].double(), s["meta"].double()
    row = 0
    for b, (n, o) in enumerate(zip(lens["new"], lens["old"])):
        x = (torch.arange(o, o + n, dtype=torch.float64, device=DEV) + c["far"])[:, None, None] * s["freqs"]
        turn = torch.polar(torch.full_like(x, s["factor"]), x)
        for name, part in (("q", s["new_q"]), ("k", s["new_k"])):
            y = part[row: row + n].double()
            z = torch.complex(y[..., 0: c["rotary"]: 2], y[..., 1: c["rotary"]: 2]) if c["inter"] else \
                torch.complex(y[..., :half], y[..., half: c["rotary"]])
            z = z * turn
            z = torch.view_as_real(z).flatten(-2) if c["inter"] else torch.cat([z.real, z.imag], -1)
            new[name].append(torch.cat([z, y[..., c["rotary"]:]], -1))
        pages = s["indices"][int(s["indptr"][b]): int(s["indptr"][b + 1])].long()
        rows = torch.arange(o, o + n, device=DEV)
        cache_k[pages[rows // PAGE], :, rows % PAGE] = new["k"][-1]
        cache_v[pages[rows // PAGE], :, rows % PAGE] = s["new_v"][row: row + n].double()
        first, last = o // PAGE, (o + n - 1) // PAGE
        for p, what in ((first, slice(o % PAGE, min(PAGE, o + n - first * PAGE))),
                        (last, slice(0, o + n - last * PAGE))):
            if p == last and last == first and what.start == 0 and o % PAGE:
                continue
            z = cache_k[pages[p], :, what]
            lo, hi = z.amin(1), z.amax(1)
            if p == first and o % PAGE:
                lo, hi = torch.minimum(lo, meta[pages[p], :, 0]), torch.maximum(hi, meta[pages[p], :, 1])
            meta[pages[p], :, 0], meta[pages[p], :, 1] = lo, hi
        whole = pages[first + 1: last]
        meta[whole, :, 0], meta[whole, :, 1] = cache_k[whole].amin(2), cache_k[whole].amax(2)
        row += n
    out = {"q": torch.cat(new["q"]), "k": cache_k, "v": cache_v, "meta": meta}
    if c["k4"]:
        out["k4"] = None  # codes are whole numbers of rounded values: no 64-bit value to come near to
    return out


def _dense(pool, ptr, indices, b, tokens, h):
    pages = indices[int(ptr[b]): int(ptr[b + 1])].long()
    return pool[pages, h].reshape(-1, D)[:tokens].double()


def _softmax64(q, k, v, keep=None):
    if not k.shape[0]:
        return torch.zeros_like(q)
    x = q @ k.T / math.sqrt(D)
    if keep is not None:
        x = x.masked_fill(~keep, -math.inf)
    return torch.softmax(x, -1) @ v


def _prefix64(s):
    c, lens = s["case"], s["lens"]
    g = c["hq"] // c["hkv"]
    out = torch.zeros(c["batch"], c["hq"], D, dtype=torch.float64, device=DEV)
    for i in range(c["groups"]):
        for h in range(c["hkv"]):
            kp, vp = (_dense(s[x], s["p_indptr"], s["p_indices"], i, lens["prefix"][i], h) for x in "kv")
            a, b = lens["group"][i], lens["group"][i + 1]
            q = s["q"][a:b, h * g: (h + 1) * g].double()
            shared = q @ kp.T / math.sqrt(D)
            for j in range(a, b):
                k, v = (_dense(s[x], s["indptr"], s["indices"], j, lens["own"][j], h) for x in "kv")
                x = torch.cat([shared[j - a], q[j - a] @ k.T / math.sqrt(D)], -1)
                p = torch.softmax(x, -1)
                n = kp.shape[0]
                out[j, h * g: (h + 1) * g] = p[:, :n] @ vp + p[:, n:] @ v
    return out


def _prompt64(s):
    c, lens = s["case"], s["lens"]
    g, block = c["hq"] // c["hkv"], c["block"]
    k_best = max(1, c["budget"] // PAGE) + (c["budget"] % PAGE != 0)
    out = torch.zeros(sum(lens["new"]), c["hq"], D, dtype=torch.float64, device=DEV)
    row = 0
    for b, (n, o) in enumerate(zip(lens["new"], lens["old"])):
        pages = s["indices"][int(s["indptr"][b]): int(s["indptr"][b + 1])].long()
        at = torch.arange(n + o, device=DEV)
        for h in range(c["hkv"]):
            k, v = (_dense(s[x], s["indptr"], s["indices"], b, n + o, h) for x in "kv")
            lo, hi = s["meta"][pages, h, 0].double(), s["meta"][pages, h, 1].double()
            wide = block * 16 if not c["budget"] else block
            for t in range(0, n, wide):
                m = min(wide, n - t)
                q = s["q"][row + t: row + t + m, h * g: (h + 1) * g].double()
                keep = at <= (torch.arange(o + t, o + t + m, device=DEV)[:, None, None])
                if c["budget"]:
                    before = (o + t) // PAGE
                    low, high = q.clamp(max=0).sum((0, 1)), q.clamp(min=0).sum((0, 1))
                    score = (low * lo[:before] + high * hi[:before]).sum(-1)
                    mine = at // PAGE >= before
                    if before:
                        best = score.sort(stable=True, dim=-1, descending=True).indices[:k_best]
                        mine |= torch.isin(at // PAGE, best)
                    keep = keep & mine
                x = _softmax64(q.flatten(0, 1), k, v, keep.expand(m, g, n + o).flatten(0, 1))
                out[row + t: row + t + m, h * g: (h + 1) * g] = x.unflatten(0, (m, g))
        row += n
    return out
