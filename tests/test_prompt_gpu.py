"""Attention of ragged prompts (dense, and over selected pages) and of decode batches with a shared prefix, against plain
64-bit implementations."""
import math

import pytest
import torch

from twilight_b200.cache import PAGE, PagedKVCache
from twilight_b200.kernel import ops

pytestmark = pytest.mark.gpu
DEV, D = "cuda", 128
SCALE = 1.0 / math.sqrt(D)
I32 = dict(dtype=torch.int32, device=DEV)


def tol_of(dtype, p, v, ref):
    """Bound on |out - ref| per element: the output's rounding (half a step), the weights' rounding (half a step of each,
    which adds up to at most eps/2 * sum p|v|), and 32-bit arithmetic over the row (2^-18 of sum p|v| covers logits up to
    64 in size, whose 32-bit products and scaled differences are off by 64 * 2^-24, and the sums)."""
    eps = torch.finfo(dtype).eps
    mass = p @ v.abs()
    return eps / 2 * ref.abs() + (eps / 2 + 2.0 ** -18) * mass + torch.finfo(dtype).smallest_normal * eps


def attend64(q, k, v, keep, scale=SCALE):
    """q [R,D], k/v [L,D], keep [R,L] -> out, lse, p in 64 bits; rows without keys give zeros and -inf."""
    x = (q @ k.T) * scale
    x = x.masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(x, -1) if k.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    return p @ v, lse, p


def pool(pages, hkv, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lean = torch.randn(hkv, 1, D, generator=g, device=DEV)
    heavy = torch.rand(pages, hkv, PAGE, 1, generator=g, device=DEV) < 0.02
    k = (torch.randn(pages, hkv, PAGE, D, generator=g, device=DEV) + (0.1 + 0.6 * heavy) * lean).to(dtype)
    v = torch.randn(pages, hkv, PAGE, D, generator=g, device=DEV).to(dtype)
    return k, v, lean, g


def table(lens, seed, at=0, total=None):
    n = [(x + PAGE - 1) // PAGE for x in lens]
    ptr = torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), **I32)
    order = torch.randperm(total or sum(n), generator=torch.Generator().manual_seed(seed))[at: at + sum(n)]
    last = torch.tensor([(x - 1) % PAGE + 1 if x else 0 for x in lens], **I32)
    return ptr, order.to(**I32), last


def dense(pages, ptr, idx, b, n, h):
    ids = idx[int(ptr[b]): int(ptr[b + 1])].long()
    return pages[ids, h].reshape(-1, D)[:n].double()


def poison_tails(k, v, ptr, idx, lens):
    """Whatever lies behind a sequence's end in its last page must not matter."""
    for b, n in enumerate(lens):
        if n % PAGE:
            page = int(idx[int(ptr[b + 1]) - 1])
            k[page, :, n % PAGE:] = float("nan")
            v[page, :, n % PAGE:] = float("inf")


def make_prompt(new, old, hq, hkv, dtype, seed=0, strided=False):
    lens = [a + b for a, b in zip(new, old)]
    ptr, idx, last = table(lens, seed + 1)
    k, v, lean, g = pool(max(1, idx.numel()), hkv, dtype, seed)
    q = torch.randn(sum(new), hkv, hq // hkv, D, generator=g, device=DEV) + 0.3 * lean
    q = q.reshape(sum(new), hq, D).to(dtype)
    if strided:  # a part of a wider projection
        wide = torch.randn(sum(new), hq + 3, D, generator=g, device=DEV).to(dtype)
        wide[:, :hq] = q
        q = wide[:, :hq]
    qo = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), **I32)
    return q, k, v, qo, (ptr, idx, last), lens


def check_prompt(q, k, v, qo, tab, lens, out, lse, causal=True, pages_of=None, block=64):
    hq, hkv, dtype = q.shape[1], k.shape[1], q.dtype
    g = hq // hkv
    for b, n in enumerate(lens):
        a, e = int(qo[b]), int(qo[b + 1])
        m = e - a
        if m == 0:
            continue
        at = torch.arange(n, device=DEV)
        where = n - m + torch.arange(m, device=DEV)
        for h in range(hkv):
            kk, vv = (dense(x, tab[0], tab[1], b, n, h) for x in (k, v))
            keep = (at <= where[:, None]) if causal else torch.ones(m, n, dtype=torch.bool, device=DEV)
            if pages_of is not None:
                allowed = torch.zeros(m, n, dtype=torch.bool, device=DEV)
                for t0 in range(0, m, block):
                    allowed[t0: t0 + block] = torch.isin(at // PAGE, pages_of(b, t0 // block, h))
                keep = keep & allowed
            keep = keep[:, None].expand(m, g, n).reshape(m * g, n)
            ref, ref_lse, p = attend64(q[a:e, h * g: (h + 1) * g].double().reshape(m * g, D), kk, vv, keep)
            got = out[a:e, h * g: (h + 1) * g].double().reshape(m * g, D)
            bad = (got - ref).abs() > tol_of(dtype, p, vv, ref)
            assert not bad.any(), (b, h, int(bad.sum()), float((got - ref).abs().max()))
            got_lse = lse[a:e, h * g: (h + 1) * g].double().reshape(-1)
            none = ref_lse == -math.inf
            assert (got_lse[none] == -math.inf).all() and not got[none].any()
            # 32-bit logits and sums: 2^-18 absolute for logits up to 64, 2^-22 of the logarithm itself
            assert ((got_lse - ref_lse)[~none].abs() <= 2.0 ** -18 + 2.0 ** -22 * ref_lse[~none].abs()).all()


PROMPTS = [
    # new, old, hq, hkv, dtype
    ([1], [0], 4, 1, torch.bfloat16),
    ([1, 1, 1], [0, 15, 16], 8, 8, torch.float16),
    ([3, 0, 17, 5], [0, 40, 0, 300], 8, 2, torch.bfloat16),
    ([64, 1, 2], [64, 1000, 0], 7, 1, torch.float16),
    ([129, 33, 300], [1, 0, 77], 6, 2, torch.bfloat16),
    ([1000], [24], 4, 4, torch.float16),
    ([257, 255], [0, 513], 16, 2, torch.bfloat16),
    ([40, 3], [2500, 4000], 5, 1, torch.bfloat16),
    ([2, 70], [31, 9], 48, 2, torch.float16),
    ([600], [0], 40, 8, torch.bfloat16),
]


@pytest.mark.parametrize("case", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attention(case, causal):
    new, old, hq, hkv, dtype = case
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=len(new), strided=sum(new) % 2 == 0)
    poison_tails(k, v, tab[0], tab[1], lens)
    status = torch.zeros(1, **I32)
    out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=max((n + 15) // 16 for n in lens), causal=causal, lse=True,
                               status=status)
    assert int(status) == 0
    k, v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    check_prompt(q, k, v, qo, tab, lens, out, lse, causal)


SPARSE = [
    # new, old, hq, hkv, dtype, budget, block
    ([200], [1000], 8, 2, torch.bfloat16, 256, 64),
    ([130, 1, 64], [37, 700, 0], 4, 4, torch.float16, 100, 32),
    ([300, 20], [5, 2000], 16, 2, torch.bfloat16, 64, 128),
    ([513], [511], 7, 1, torch.float16, 17, 16),
    ([100, 90], [0, 3000], 6, 2, torch.bfloat16, 5000, 64),      # the budget covers everything
    ([2, 3, 1], [900, 0, 1500], 8, 1, torch.bfloat16, 128, 64),  # a few tokens each
]


def plain_blocks(q, meta, qo, tab, lens, budget, block, b, j, h, g):
    """Pages of block j of sequence b for KV head h, and the history's scores, in 64 bits."""
    a, e = int(qo[b]), int(qo[b + 1])
    t0 = j * block
    rows = q[a + t0: min(e, a + t0 + block), h * g: (h + 1) * g].double().reshape(-1, D)
    first = lens[b] - (e - a) + t0
    last = first + rows.shape[0] // g - 1
    n = first // PAGE
    ids = tab[1][int(tab[0][b]): int(tab[0][b + 1])].long()[:n]
    lo, hi = meta[ids, h, 0].double(), meta[ids, h, 1].double()
    score = torch.maximum(rows[:, None] * lo, rows[:, None] * hi).sum((0, 2)) if n else torch.zeros(0, device=DEV)
    k = max(1, budget // PAGE) + (budget % PAGE != 0)
    return score, min(k, n), torch.arange(n, last // PAGE + 1, device=DEV), rows


@pytest.mark.parametrize("case", SPARSE, ids=[str(i) for i in range(len(SPARSE))])
def test_selected_pages_and_sparse_prompt_attention(case):
    new, old, hq, hkv, dtype, budget, block = case
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=7)
    g = hq // hkv
    most = max((n + 15) // 16 for n in lens)
    meta = ops.build_page_meta(k, *tab, max_pages=most)
    poison_tails(k, v, tab[0], tab[1], lens)
    status = torch.zeros(1, **I32)
    pages, count = ops.quest_select_blocks(q, meta, qo, *tab, budget, max_pages=most, query_block=block, status=status)
    assert int(status) == 0

    def slot(b, j):
        return int(qo[b]) // block + b + j

    for b in range(len(new)):
        for j in range((new[b] + block - 1) // block):
            for h in range(hkv):
                got = pages[slot(b, j), h, : int(count[slot(b, j), h])].long()
                score, n, mine, rows = plain_blocks(q, meta, qo, tab, lens, budget, block, b, j, h, g)
                assert got.numel() == n + mine.numel() and (got[1:] > got[:-1]).all()
                assert torch.equal(got[n:], mine)
                if n < score.numel():  # a 32-bit sum of rows*256 products: near ties may go either way
                    cut = score.sort(descending=True).values[n - 1]
                    off = 2.0 ** -20 * (rows.abs().sum(0) * meta.double().abs().amax()).sum()
                    chosen = torch.zeros_like(score, dtype=torch.bool)
                    chosen[got[:n]] = True
                    assert chosen[score > cut + off].all() and not chosen[score < cut - off].any()
    out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=most, block_pages=pages, block_npages=count,
                               query_block=block, lse=True, status=status)
    assert int(status) == 0
    k, v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    check_prompt(q, k, v, qo, tab, lens, out, lse, True,
                 lambda b, j, h: pages[slot(b, j), h, : int(count[slot(b, j), h])], block)


def test_lists_of_a_caller_empty_rows_and_bad_pages():
    new, old = [70, 40], [100, 10]
    q, k, v, qo, tab, lens = make_prompt(new, old, 4, 2, torch.bfloat16, seed=3)
    block, slots = 32, sum(new) // 32 + 2
    pages = torch.full((slots, 2, 5), -7, **I32)
    count = torch.zeros(slots, 2, **I32)
    # block 0 of sequence 0: page 1 only; block 1: nothing; block 2: only a page behind all its queries but the last ones
    pages[0, :, 0], count[0] = 1, 1
    pages[2, :, 0], count[2] = 10, 1
    first = 110 // 32 * 0 + int(qo[1]) // block + 1
    pages[first, :, :2], count[first] = torch.tensor([0, 2], **I32), 2
    pages[first + 1, :, :1], count[first + 1] = torch.tensor([3], **I32), 1
    status = torch.zeros(1, **I32)
    out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=11, block_pages=pages, block_npages=count,
                               query_block=block, lse=True, status=status)
    assert int(status) == 0
    base = [0, first]
    check_prompt(q, k, v, qo, tab, lens, out, lse, True, lambda b, j, h: pages[base[b] + j, h, : int(count[base[b] + j, h])],
                 block)
    assert not out[32:64].any() and (lse[32:64] == -math.inf).all()
    # a page that is not there is skipped and flagged
    pages[0, :, 1], count[0] = 500, 2
    got = ops.prompt_attn(q, k, v, qo, *tab, max_pages=11, block_pages=pages, block_npages=count, query_block=block,
                          status=status)
    assert int(status) == ops.FLAG_BAD_INDEX and torch.equal(got, out)
    status.zero_()
    idx = tab[1].clone()
    idx[1] = -1
    ops.prompt_attn(q, k, v, qo, tab[0], idx, tab[2], max_pages=11, status=status)
    assert int(status) == ops.FLAG_BAD_INDEX


def test_rows_behind_the_last_sequence_are_left_and_extreme_logits():
    q, k, v, qo, tab, lens = make_prompt([20, 30], [0, 200], 4, 2, torch.bfloat16, seed=5)
    out = torch.full_like(q, 7.0)
    short = qo.clone()
    short[2] = 41
    # the second sequence then has 21 new tokens, its last ones
    ops.prompt_attn(q, k, v, short, *tab, max_pages=15, out=out)
    assert (out[41:] == 7.0).all() and not (out[:41] == 7.0).all(-1).any()
    # logits of +-1000: the softmax is one key's, or an even split between equal ones
    q2 = torch.zeros_like(q)
    q2[:, :, 0] = 100.0
    k2 = torch.zeros_like(k)
    k2[..., 0] = -100.0
    page = int(tab[1][0])
    k2[page, :, 3, 0] = 100.0
    got = ops.prompt_attn(q2, k2, v, qo, *tab, max_pages=15)
    want = v[page, :, 3].repeat_interleave(2, 0)
    assert torch.equal(got[5:20], want.expand(15, 4, D))
    assert torch.isfinite(got.float()).all()


PREFIXES = [
    # group sizes, prefix lengths, own lengths (cycled), hq, hkv, dtype
    ([1], [0], [0], 4, 1, torch.bfloat16),
    ([2, 1], [40, 0], [0, 17, 0], 8, 2, torch.float16),
    ([3, 5], [1, 300], [0, 1, 16, 33], 8, 8, torch.bfloat16),
    ([40], [1000], [5, 0, 130], 8, 2, torch.bfloat16),
    ([7, 33, 1], [129, 2047, 16], [700, 3], 7, 1, torch.float16),
    ([150], [777], [1], 16, 2, torch.bfloat16),
    ([20, 0, 13], [100, 50, 4100], [64, 65, 0], 40, 8, torch.bfloat16),
    ([70], [5000], [20], 32, 1, torch.float16),
    ([300], [513], [0, 40], 4, 4, torch.float16),
]


@pytest.mark.parametrize("case", PREFIXES, ids=[str(i) for i in range(len(PREFIXES))])
def test_shared_prefix_attention(case):
    sizes, prefix, own, hq, hkv, dtype = case
    n = sum(sizes)
    own = [own[i % len(own)] for i in range(n)]
    pages = sum((x + 15) // 16 for x in prefix + own)
    total = max(pages, 1)
    ptr, idx, last = table(own, 4, 0, total)
    pptr, pidx, plast = table(prefix, 4, idx.numel(), total)
    k, v, lean, g = pool(total, hkv, dtype, 9)
    q = (torch.randn(n, hkv, hq // hkv, D, generator=g, device=DEV) + 0.3 * lean).reshape(n, hq, D).to(dtype)
    poison_tails(k, v, ptr, idx, own)
    poison_tails(k, v, pptr, pidx, prefix)
    group = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), **I32)
    status = torch.zeros(1, **I32)
    args = (q, k, v, group, pptr, pidx, plast, ptr, idx, last)
    out, lse = ops.shared_prefix_attn(*args, lse=True, status=status)
    assert int(status) == 0
    most = max(1, max((x + 15) // 16 for x in prefix + own))
    again = ops.shared_prefix_attn(*args[:1], *args[1:], max_pages=most)
    assert torch.equal(again, out)                              # the same with the exact bound, and twice
    k, v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    gq = hq // hkv
    for i in range(len(sizes)):
        for b in range(int(group[i]), int(group[i + 1])):
            for h in range(hkv):
                kk = torch.cat([dense(k, pptr, pidx, i, prefix[i], h), dense(k, ptr, idx, b, own[b], h)])
                vv = torch.cat([dense(v, pptr, pidx, i, prefix[i], h), dense(v, ptr, idx, b, own[b], h)])
                keep = torch.ones(gq, kk.shape[0], dtype=torch.bool, device=DEV)
                ref, ref_lse, p = attend64(q[b, h * gq: (h + 1) * gq].double(), kk, vv, keep)
                got = out[b, h * gq: (h + 1) * gq].double()
                assert ((got - ref).abs() <= tol_of(dtype, p, vv, ref)).all(), (i, b, h, float((got - ref).abs().max()))
                got_lse = lse[b, h * gq: (h + 1) * gq].double()
                if kk.shape[0] == 0:
                    assert (got_lse == -math.inf).all() and not got.any()
                else:
                    assert ((got_lse - ref_lse).abs() <= 2.0 ** -18 + 2.0 ** -22 * ref_lse.abs()).all()


def test_a_sequence_in_no_group_has_no_prefix():
    own = [20, 30, 5]
    ptr, idx, last = table(own + [64], 2)
    k, v, lean, g = pool(idx.numel(), 2, torch.bfloat16, 1)
    q = torch.randn(3, 4, D, generator=g, device=DEV).to(torch.bfloat16)
    pptr, pidx, plast = torch.tensor([0, 4], **I32), idx[-4:].contiguous(), torch.tensor([16], **I32)
    args = (ptr[:4].contiguous(), idx, last[:3].contiguous())
    got = ops.shared_prefix_attn(q, k, v, torch.tensor([1, 2], **I32), pptr, pidx, plast, *args)
    alone = ops.prompt_attn(q, k, v, torch.arange(4, **I32), *args, max_pages=2)
    all_in = ops.shared_prefix_attn(q, k, v, torch.tensor([0, 3], **I32), pptr, pidx, plast, *args)
    for b, want in ((0, alone), (1, all_in), (2, alone)):
        assert (got[b].float() - want[b].float()).abs().max() <= 2.0 ** -7 * want[b].float().abs().max()


def test_graph_side_stream_and_a_workspace_of_the_callers():
    q, k, v, qo, tab, lens = make_prompt([300, 40], [500, 0], 8, 2, torch.bfloat16, seed=2)
    want = ops.prompt_attn(q, k, v, qo, *tab, max_pages=50)
    ws = torch.full((ops.prompt_attn_workspace_bytes(340, 2, 8, 2, 50),), 255, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(want)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        ops.prompt_attn(q, k, v, qo, *tab, max_pages=50, out=out, workspace=ws)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_prompts_whole_way_through_the_operators():
    """Append with rotation, select, attend in two chunks; then a decode step over the prompt as a shared prefix.  The
    same prompt in one chunk gives the same, within what rounding twice allows."""
    hq, hkv, dtype, n = 8, 2, torch.bfloat16, 700
    g = torch.Generator(device=DEV).manual_seed(11)
    proj = torch.randn(n, hq + 2 * hkv, D, generator=g, device=DEV).to(dtype)
    parts = proj[:, :hq], proj[:, hq: hq + hkv], proj[:, hq + hkv:]
    freqs, scale = ops.rope_frequencies(D, 500000.0, device=DEV)
    ptr, idx, last = table([n], 5)
    results = []
    for cuts in ([0, n], [0, 400, n]):
        k, v = (torch.zeros(idx.numel(), hkv, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
        k4 = torch.zeros(idx.numel(), hkv, 1280, dtype=torch.uint8, device=DEV)
        meta = torch.zeros(idx.numel(), hkv, 2, D, dtype=dtype, device=DEV)
        outs = []
        for a, e in zip(cuts, cuts[1:]):
            p1, i1, l1 = PagedKVCache.page_table([e], DEV)[:3]
            tab = (p1, idx[: p1[-1]].contiguous(), l1)
            qo = torch.tensor([0, e - a], **I32)
            q = ops.rope_append_kv(*(x[a:e] for x in parts), freqs, k, v, k4, meta, qo, *tab, attention_scale=scale)
            sel = ops.quest_select_blocks(q, meta, qo, *tab, 1024, max_pages=44, query_block=16)
            outs.append(ops.prompt_attn(q, k, v, qo, *tab, max_pages=44, block_pages=sel[0], block_npages=sel[1],
                                        query_block=16))
        results.append((torch.cat(outs), k, v, k4, meta))
    for a, b in zip(results[0][1:], results[1][1:]):
        assert torch.equal(a, b)
    x, y = results[0][0].float(), results[1][0].float()
    assert ((x - y).abs() <= 2.0 ** -7 * y.abs() + 2.0 ** -7 * v.float().abs().max()).all()
    k, v = results[0][1:3]
    qd = torch.randn(3, hq, D, generator=g, device=DEV).to(dtype)
    none = torch.zeros(4, **I32), torch.zeros(0, **I32), torch.zeros(3, **I32)
    got = ops.shared_prefix_attn(qd, k, v, torch.tensor([0, 3], **I32), ptr, idx, last, *none)
    kk, vv = (dense(x, ptr, idx, 0, n, 0) for x in (k, v))
    ref, _, p = attend64(qd[1, :4].double(), kk, vv, torch.ones(4, n, dtype=torch.bool, device=DEV))
    assert ((got[1, :4].double() - ref).abs() <= tol_of(dtype, p, vv, ref)).all()


@pytest.mark.parametrize("seed", range(10))
def test_prompt_fuzz(seed):
    """Random batches: head groupings, lengths around the tiles' and chunks' borders, both masks, lists or none."""
    r = torch.Generator().manual_seed(100 + seed)
    pick = lambda xs: xs[int(torch.randint(len(xs), (1,), generator=r))]  # noqa: E731
    for _ in range(5):
        hkv, g = pick([(1, 1), (2, 1), (1, 2), (2, 3), (1, 4), (2, 5), (1, 7), (2, 8), (1, 12), (1, 33)])
        dtype = pick([torch.float16, torch.bfloat16])
        n = pick([1, 1, 2, 5])
        new = [pick([0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 257, 300]) for _ in range(n)]
        old = [pick([0, 0, 1, 15, 16, 100, 111, 112, 127, 128, 500, 1024, 1500, 3000]) for _ in range(n)]
        if sum(new) == 0 or sum(a + b for a, b in zip(new, old)) == 0:
            continue
        q, k, v, qo, tab, lens = make_prompt(new, old, g * hkv, hkv, dtype, seed=seed)
        most = max(1, max((x + 15) // 16 for x in lens))
        block = pick([16, 32, 64, 128])
        sparse, causal = pick([False, True]), pick([True, True, False])
        kw, pages_of = {}, None
        if sparse:
            meta = ops.build_page_meta(k, *tab, max_pages=most)
            pages, count = ops.quest_select_blocks(q, meta, qo, *tab, pick([16, 100, 640]), max_pages=most, query_block=block)
            kw = dict(block_pages=pages, block_npages=count, query_block=block)

            def pages_of(b, j, h, pages=pages, count=count, qo=qo, block=block):
                s = int(qo[b]) // block + b + j
                return pages[s, h, : int(count[s, h])]
        poison_tails(k, v, tab[0], tab[1], lens)
        status = torch.zeros(1, **I32)
        out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=most, causal=causal, lse=True, status=status, **kw)
        assert int(status) == 0
        k, v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
        check_prompt(q, k, v, qo, tab, lens, out, lse, causal, pages_of, block)


@pytest.mark.parametrize("case", [
    # a few tokens over a long context: runs and chunks of the keys, joined; and many tiles over one
    ([1], [40000], 8, 1, torch.bfloat16),
    ([4], [30011], 8, 2, torch.float16),
    ([20], [30000], 8, 2, torch.bfloat16),
    ([130], [20000], 2, 2, torch.float16),
    ([700], [9000], 4, 1, torch.bfloat16),
    ([40, 1, 3], [12000, 9000, 0], 16, 2, torch.bfloat16),
])
def test_prompt_long_contexts(case):
    new, old, hq, hkv, dtype = case
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=13)
    out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=max((n + 15) // 16 for n in lens), lse=True)
    check_prompt(q, k, v, qo, tab, lens, out, lse)
    again = ops.prompt_attn(q, k, v, qo, *tab, max_pages=max((n + 15) // 16 for n in lens))
    assert torch.equal(out, again)                              # the order of the work does not show


def test_pages_behind_32_bit_offsets():
    """Pools of more than 2^32 elements, the pages in use at their end: append, selection, attention of both kinds."""
    hq, hkv, n, dtype = 16, 8, 200, torch.bfloat16
    pages = 2 ** 32 // (hkv * PAGE * D) + 64
    k, v = (torch.empty(pages, hkv, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
    meta = torch.empty(pages, hkv, 2, D, dtype=dtype, device=DEV)
    idx = (pages - 1 - torch.randperm(13)).to(**I32)
    tab = (torch.tensor([0, 13], **I32), idx, torch.tensor([8], **I32))
    g = torch.Generator(device=DEV).manual_seed(1)
    proj = torch.randn(n, hq + 2 * hkv, D, generator=g, device=DEV).to(dtype)
    qo = torch.tensor([0, n], **I32)
    q = ops.rope_append_kv(proj[:, :hq], proj[:, hq: hq + hkv], proj[:, hq + hkv:], None, k, v, None, meta, qo, *tab)
    kk = k[idx.long()].transpose(0, 1).reshape(hkv, -1, D)[:, :n]
    assert torch.equal(kk, proj[:, hq: hq + hkv].transpose(0, 1))
    lens = [n]
    sel = ops.quest_select_blocks(q, meta, qo, *tab, 64, max_pages=13, query_block=32)
    out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=13, block_pages=sel[0], block_npages=sel[1], query_block=32, lse=True)
    # (sequence 0's query block j is slot j)
    check_prompt(q, k, v, qo, tab, lens, out, lse, True, lambda b, j, h: sel[0][j, h, : int(sel[1][j, h])], 32)
    none = torch.zeros(4, **I32), torch.zeros(0, **I32), torch.zeros(3, **I32)
    got = ops.shared_prefix_attn(q[:3], k, v, torch.tensor([0, 3], **I32), *tab, *none)
    want = ops.prompt_attn(q[:3], k, v, torch.tensor([0, 3], **I32), *tab, max_pages=13, causal=False)
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


def test_a_nan_or_infinity_of_a_visible_key_shows_and_a_masked_one_does_not():
    for new, old in (([3], [60]), ([100], [60])):
        q, k, v, qo, tab, lens = make_prompt(new, old, 4, 2, torch.bfloat16, seed=4)
        clean = ops.prompt_attn(q, k, v, qo, *tab, max_pages=10)
        bad = k.clone()
        page, row = int(tab[1][(lens[0] - 1) // PAGE]), (lens[0] - 1) % PAGE
        bad[page, 0, row] = float("nan")                        # the last token's K: only the last query sees it
        got = ops.prompt_attn(q, bad, v, qo, *tab, max_pages=10)
        assert torch.isnan(got[-1, :2].float()).all()
        assert torch.equal(got[:-1], clean[:-1]) and torch.equal(got[-1, 2:], clean[-1, 2:])
        bad = k.clone()
        bad[int(tab[1][0]), 1, 5] = float("nan")                # a token that every query sees
        got = ops.prompt_attn(q, bad, v, qo, *tab, max_pages=10)
        assert torch.isnan(got[:, 2:].float()).all() and torch.equal(got[:, :2], clean[:, :2])


def test_calls_on_two_streams_and_two_graphs_with_their_own_workspaces():
    a = make_prompt([500, 3], [100, 4000], 8, 2, torch.bfloat16, seed=21)
    b = make_prompt([90], [2000], 8, 2, torch.bfloat16, seed=22)
    calls = [lambda ws=None, out=None, x=x: ops.prompt_attn(*x[:4], *x[4], max_pages=260, workspace=ws, out=out) for x in (a, b)]
    want = [f() for f in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for i, f in enumerate(calls):
        x = (a, b)[i]
        n = ops.prompt_attn_workspace_bytes(x[0].shape[0], len(x[5]), 8, 2, 260)
        ws, out = torch.empty(n, dtype=torch.uint8, device=DEV), torch.zeros_like(want[i])
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f(ws, out)
        graphs.append(gr)
        outs.append((out, ws))
    torch.cuda.synchronize()
    for s, gr in zip(streams, graphs):
        with torch.cuda.stream(s):
            for _ in range(3):
                gr.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i][0], want[i])


def test_too_small_max_pages_is_flagged_and_stays_in_its_workspace():
    q, k, v, qo, tab, lens = make_prompt([2] * 40, [3000] * 40, 8, 2, torch.bfloat16, seed=6)
    n = ops.prompt_attn_workspace_bytes(80, 40, 8, 2, 1)
    ws = torch.full((n + 4096,), 173, dtype=torch.uint8, device=DEV)
    status = torch.zeros(1, **I32)
    ops.prompt_attn(q, k, v, qo, *tab, max_pages=1, workspace=ws[:n], status=status)
    assert int(status) & ops.FLAG_BAD_INDEX and (ws[n:] == 173).all()


def test_one_token_of_a_batch_with_a_foreign_stride_and_no_pages():
    q, k, v, qo, tab, lens = make_prompt([1], [50], 4, 2, torch.float16, seed=8)
    odd = torch.as_strided(q, q.shape, (13, D, 1))              # one token: its stride means nothing
    assert torch.equal(ops.prompt_attn(odd, k, v, qo, *tab, max_pages=4), ops.prompt_attn(q, k, v, qo, *tab, max_pages=4))
    empty = torch.zeros(2, **I32), torch.zeros(0, **I32), torch.zeros(1, **I32)
    out, lse = ops.prompt_attn(q, k, v, qo, *empty, max_pages=1, lse=True)
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("seed", range(6))
def test_shared_prefix_fuzz(seed):
    r = torch.Generator().manual_seed(300 + seed)
    pick = lambda xs: xs[int(torch.randint(len(xs), (1,), generator=r))]  # noqa: E731
    for _ in range(3):
        hkv, gq = pick([(1, 1), (2, 4), (1, 8), (2, 5), (1, 16), (1, 9)])
        dtype = pick([torch.float16, torch.bfloat16])
        sizes = [pick([0, 1, 2, 3, 9, 16, 17, 60]) for _ in range(pick([1, 2, 4]))]
        n = sum(sizes)
        if n == 0:
            continue
        prefix = [pick([0, 1, 16, 127, 128, 129, 500, 2049]) for _ in sizes]
        own = [pick([0, 0, 1, 15, 16, 17, 200, 700]) for _ in range(n)]
        total = max(1, sum((x + 15) // 16 for x in prefix + own))
        ptr, idx, last = table(own, 4, 0, total)
        pptr, pidx, plast = table(prefix, 4, idx.numel(), total)
        k, v, lean, g = pool(total, hkv, dtype, seed)
        q = (torch.randn(n, hkv, gq, D, generator=g, device=DEV) + 0.3 * lean).reshape(n, hkv * gq, D).to(dtype)
        poison_tails(k, v, ptr, idx, own)
        poison_tails(k, v, pptr, pidx, prefix)
        group = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), **I32)
        out = ops.shared_prefix_attn(q, k, v, group, pptr, pidx, plast, ptr, idx, last)
        k, v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
        for i in range(len(sizes)):
            for b in range(int(group[i]), int(group[i + 1])):
                for h in range(hkv):
                    kk = torch.cat([dense(k, pptr, pidx, i, prefix[i], h), dense(k, ptr, idx, b, own[b], h)])
                    vv = torch.cat([dense(v, pptr, pidx, i, prefix[i], h), dense(v, ptr, idx, b, own[b], h)])
                    ref, _, p = attend64(q[b, h * gq: (h + 1) * gq].double(), kk, vv,
                                         torch.ones(gq, kk.shape[0], dtype=torch.bool, device=DEV))
                    got = out[b, h * gq: (h + 1) * gq].double()
                    assert ((got - ref).abs() <= tol_of(dtype, p, vv, ref)).all(), (sizes, prefix, i, b, h)


@pytest.mark.parametrize("case", [
    # more tiles than blocks, by a few
    ([5200], [1000], 8, 8, torch.bfloat16, 0),
    ([5000], [3000], 32, 8, torch.float16, 0),
    ([1300, 1301], [2000, 2500], 32, 8, torch.bfloat16, 512),
    ([2400, 9], [4000, 0], 64, 8, torch.bfloat16, 640),
])
def test_partly_filled_waves_of_tiles(case):
    new, old, hq, hkv, dtype, budget = case
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=17)
    most = max((n + 15) // 16 for n in lens)
    kw, pages_of = {}, None
    if budget:
        meta = ops.build_page_meta(k, *tab, max_pages=most)
        pages, count = ops.quest_select_blocks(q, meta, qo, *tab, budget, max_pages=most, query_block=64)
        kw = dict(block_pages=pages, block_npages=count, query_block=64)

        def pages_of(b, j, h):
            s = int(qo[b]) // 64 + b + j
            return pages[s, h, : int(count[s, h])]
    for causal in (True, False):
        status = torch.zeros(1, **I32)
        out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=most, causal=causal, lse=True, status=status, **kw)
        assert int(status) == 0
        check_prompt(q, k, v, qo, tab, lens, out, lse, causal, pages_of, 64)


def test_many_sequences_over_one_prefix():
    n, hq, hkv, prefix = 640, 64, 8, 3000
    ptr, idx, last = torch.zeros(n + 1, **I32), torch.zeros(0, **I32), torch.zeros(n, **I32)
    pptr, pidx, plast = table([prefix], 1)
    k, v, lean, g = pool(pidx.numel(), hkv, torch.bfloat16, 2)
    q = (torch.randn(n, hkv, hq // hkv, D, generator=g, device=DEV) + 0.3 * lean).reshape(n, hq, D).to(torch.bfloat16)
    status = torch.zeros(1, **I32)
    out, lse = ops.shared_prefix_attn(q, k, v, torch.tensor([0, n], **I32), pptr, pidx, plast, ptr, idx, last, lse=True,
                                      max_pages=(prefix + 15) // 16, status=status)
    assert int(status) == 0
    check_prompt(q, k, v, torch.tensor([0, n], **I32), (pptr, pidx, plast), [prefix], out, lse, causal=False)


@pytest.mark.parametrize("lead", [1, 64, 161])
def test_a_part_of_a_larger_batch(lead):
    """Offsets that begin behind row 0: the results of the part alone, and rows of no sequence are left."""
    new, old, hq, hkv = [70, 1, 130], [300, 900, 0], 8, 2
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, torch.bfloat16, seed=11)
    meta = torch.stack([k.amin(2), k.amax(2)], 2).contiguous()
    most = max((n + 15) // 16 for n in lens)
    wide = torch.nn.functional.pad(q, (0, 0, 0, 0, lead, 9), value=3.0)
    t = q.shape[0]
    for block in (None, 32):
        args, wargs = {}, {}
        if block:
            pages, counts = ops.quest_select_blocks(q, meta, qo, *tab, 128, max_pages=most, query_block=block)
            args = dict(block_pages=pages, block_npages=counts, query_block=block)
            wpages, wcounts = ops.quest_select_blocks(wide, meta, qo + lead, *tab, 128, max_pages=most, query_block=block)
            wargs = dict(block_pages=wpages, block_npages=wcounts, query_block=block)
            for b, n in enumerate(new):
                for j in range((n + block - 1) // block):
                    one = int(qo[b]) // block + b + j
                    two = (int(qo[b]) + lead) // block + b + j
                    assert torch.equal(counts[one], wcounts[two])
                    for h in range(hkv):
                        c = int(counts[one, h])
                        assert torch.equal(pages[one, h, :c], wpages[two, h, :c])
        want = ops.prompt_attn(q, k, v, qo, *tab, max_pages=most, **args)
        out = torch.full_like(wide, 5.0)
        status = torch.zeros(1, **I32)
        ops.prompt_attn(wide, k, v, qo + lead, *tab, max_pages=most, out=out, status=status, **wargs)
        assert int(status) == 0 and torch.equal(out[lead: lead + t], want)
        assert (out[:lead] == 5).all() and (out[lead + t:] == 5).all()


def test_calls_one_after_another_see_what_was_written_before_each():
    """A long chunk, a few tokens and many single ones in one call (both attention kernels have work), over and over, with
    queries, pages, page table and lengths rewritten by kernels right before each call: the same as with the GPU waited for."""
    new = [300, 5] + [1] * 60
    old = [900, 40] + [37 * i % 700 for i in range(60)]
    rounds = []
    for i in range(6):
        shift = [max(0, x - 16 * i) for x in old]
        rounds.append(make_prompt(new, shift, 8, 2, torch.bfloat16, seed=30 + i))
    pages = max(r[1].shape[0] for r in rounds)
    entries = max(r[4][1].numel() for r in rounds)
    q, qo = torch.empty_like(rounds[0][0]), rounds[0][3]
    k, v = (torch.empty(pages, 2, PAGE, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ptr, idx, last = torch.empty(63, **I32), torch.empty(entries, **I32), torch.empty(62, **I32)
    ws = torch.empty(ops.prompt_attn_workspace_bytes(q.shape[0], 62, 8, 2, 80), dtype=torch.uint8, device=DEV)

    def one(r, wait):
        x, kk, vv, _, tab, _ = r
        for to, of in ((q, x), (k[: kk.shape[0]], kk), (v[: vv.shape[0]], vv), (ptr, tab[0]), (idx[: tab[1].numel()], tab[1]),
                       (last, tab[2])):
            to.copy_(of)
        if wait:
            torch.cuda.synchronize()
        out = ops.prompt_attn(q, k, v, qo, ptr, idx, last, max_pages=80, workspace=ws)
        if wait:
            torch.cuda.synchronize()
        return out

    want = [one(r, True) for r in rounds]
    got = [one(r, False) for r in rounds * 4]
    assert all(torch.equal(x, want[i % 6]) for i, x in enumerate(got))
    x, kk, vv, qo, tab, lens = rounds[-1]
    out, lse = ops.prompt_attn(x, kk, vv, qo, *tab, max_pages=80, lse=True)
    check_prompt(x, kk, vv, qo, tab, lens, out, lse)


def block_sums64(q, meta, qo, tab, lens, block, b, j, hkv):
    """Scores of the pages before block j of sequence b in 64 bits, [pages, hkv], and the sums of their parts' sizes."""
    a, e = int(qo[b]), int(qo[b + 1])
    rows = q[a + j * block: min(e, a + (j + 1) * block)].double().unflatten(1, (hkv, -1))
    n = (lens[b] - (e - a) + j * block) // PAGE
    ids = tab[1][int(tab[0][b]): int(tab[0][b + 1])].long()[:n]
    low, high = rows.clamp(max=0).sum((0, 2)), rows.clamp(min=0).sum((0, 2))
    lo, hi = low * meta[ids, :, 0].double(), high * meta[ids, :, 1].double()
    return (lo + hi).sum(-1), (lo.abs() + hi.abs()).sum(-1), rows.shape[0] * rows.shape[2]


@pytest.mark.parametrize("scale", [1.0, 1e-2, 1e-4, 1e-5])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_scores_are_32_bit_sums_whatever_the_queries_size(dtype, scale):
    new, old, hq, hkv, block = [128, 90], [1000, 2500], 8, 2, 32
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=40)
    q = (q.float() * scale).to(dtype)
    most = max((n + 15) // 16 for n in lens)
    meta = ops.build_page_meta(k, *tab, max_pages=most)
    slots = sum(new) // block + len(new)
    scores = torch.zeros(slots, hkv, most, device=DEV)
    ops.quest_select_blocks(q, meta, qo, *tab, 256, max_pages=most, query_block=block, page_scores=scores)
    for b in range(len(new)):
        for j in range((new[b] + block - 1) // block):
            want, size, rows = block_sums64(q, meta, qo, tab, lens, block, b, j, hkv)
            got = scores[int(qo[b]) // block + b + j, :, : want.shape[0]].T.double()
            # In steps of 2^-24 of the sum of the parts' sizes: the pooled sums in 16 runs (rows/16 + 15 roundings, of numbers of
            # one sign), their parts (4: 22 bits), tensor-core sums of 16 products and what they are added to (17 numbers cut off
            # below 2 steps each, twice for every 32 numbers), sums of those (8)
            assert ((got - want).abs() <= (rows / 16 + 15 + 4 + 68 + 8) * 2.0 ** -24 * size).all()


def exact_lists(q, meta, qo, tab, lens, budget, block, hkv, got, count):
    """Compares block lists with the 64-bit choice, ties to the lower page; the number of lists that had a choice."""
    k = max(1, budget // PAGE) + (budget % PAGE != 0)
    lists = 0
    for b, total in enumerate(lens):
        m = int(qo[b + 1]) - int(qo[b])
        for j in range((m + block - 1) // block):
            want = block_sums64(q, meta, qo, tab, lens, block, b, j, hkv)[0]
            n, slot = want.shape[0], int(qo[b]) // block + b + j
            best = want.sort(dim=0, stable=True, descending=True).indices[:k].sort(dim=0).values
            assert torch.equal(got[slot, :, : min(k, n)].long().T, best), (b, j)
            own = torch.arange(n, (total - m + min(m, (j + 1) * block) - 1) // PAGE + 1, device=DEV)
            assert (count[slot] == best.shape[0] + own.shape[0]).all()
            assert (got[slot, :, best.shape[0]: best.shape[0] + own.shape[0]] == own).all()
            lists += hkv * (n > k)
    return lists


@pytest.mark.parametrize("case", [
    # new, old, hq, hkv, budget, block, scale
    ([1500, 700], [4000, 9000], 8, 8, 1024, 128, 1.0),
    ([1500, 700], [4000, 9000], 16, 4, 4096, 64, 1.0),
    ([700, 300], [4000, 2000], 8, 8, 1024, 64, 1e-3),
    ([700, 300], [4000, 2000], 8, 8, 1024, 64, 1e-4),
    ([40], [20000], 48, 1, 100, 16, 1e-2),
], ids=[str(i) for i in range(5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chosen_pages_are_those_of_the_64_bit_sums(dtype, case):
    new, old, hq, hkv, budget, block, scale = case
    for seed in range(3):
        q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=50 + seed)
        q = (q.float() * scale).to(dtype)
        most = max((n + 15) // 16 for n in lens)
        meta = ops.build_page_meta(k, *tab, max_pages=most)
        status = torch.zeros(1, **I32)
        pages, count = ops.quest_select_blocks(q, meta, qo, *tab, budget, max_pages=most, query_block=block, status=status)
        assert int(status) == 0
        assert exact_lists(q, meta, qo, tab, lens, budget, block, hkv, pages, count) > 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spread", ["one step in a few channels", "none", "no queries", "one page apart"])
def test_chosen_pages_among_near_and_equal_scores(dtype, spread):
    """Every page has (nearly) the same metadata: the cut lies among scores that 32 bits do not tell apart, or among equal ones,
    where the lower page goes first."""
    new, old, hq, hkv, budget, block = [70, 33], [3000, 5000], 4, 2, 700, 32
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=60)
    g = torch.Generator(device=DEV).manual_seed(61)
    most = max((n + 15) // 16 for n in lens)
    pages = k.shape[0]
    base = torch.randn(1, hkv, 2, D, generator=g, device=DEV).abs()
    base[:, :, 0] *= -1
    meta = base.to(dtype).repeat(pages, 1, 1, 1).contiguous()
    if spread == "one step in a few channels":
        bits = meta.view(torch.int16)
        some = torch.rand(meta.shape, generator=g, device=DEV) < 0.05
        bits += some * torch.randint(-1, 2, meta.shape, generator=g, device=DEV, dtype=torch.int16)
    if spread == "one page apart":
        meta[int(tab[1][77])] *= 2.0
    if spread == "no queries":
        q = torch.zeros_like(q)
    got = ops.quest_select_blocks(q, meta, qo, *tab, budget, max_pages=most, query_block=block)
    assert exact_lists(q, meta, qo, tab, lens, budget, block, hkv, *got) > 0


def test_sparse_prompts_against_the_definition():
    """Selection and attention together, by the definition's own choice of pages."""
    for new, old, hq, hkv, dtype, budget, block in (([500, 300], [2000, 100], 4, 4, torch.float16, 512, 128),
                                                    ([260], [4000], 8, 2, torch.bfloat16, 1024, 64)):
        q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, dtype, seed=70)
        most = max((n + 15) // 16 for n in lens)
        meta = ops.build_page_meta(k, *tab, max_pages=most)
        sel = ops.quest_select_blocks(q, meta, qo, *tab, budget, max_pages=most, query_block=block)
        out, lse = ops.prompt_attn(q, k, v, qo, *tab, max_pages=most, block_pages=sel[0], block_npages=sel[1],
                                   query_block=block, lse=True)

        def pages_of(b, j, h):
            want = block_sums64(q, meta, qo, tab, lens, block, b, j, hkv)[0][:, h]
            best = want.sort(stable=True, descending=True).indices[: max(1, budget // PAGE) + (budget % PAGE != 0)]
            return torch.cat([best, torch.arange(want.shape[0], most, device=DEV)])

        check_prompt(q, k, v, qo, tab, lens, out, lse, True, pages_of, block)


@pytest.mark.parametrize("heads", [(33, 1), (48, 1), (128, 2), (128, 1)])
@pytest.mark.parametrize("batch", [1, 2, 3, 260])
def test_shared_prefix_of_many_query_heads(heads, batch):
    """A sequence's own part alone is more rows than the row kernel takes: both parts leave partial results of the tile kernel."""
    hq, hkv = heads
    own, prefix = [(1 + 13 * i) % 64 for i in range(batch)], [60]
    total = sum((x + 15) // 16 for x in own + prefix)
    ptr, idx, last = table(own, 4, 0, total)
    pptr, pidx, plast = table(prefix, 4, idx.numel(), total)
    k, v, lean, g = pool(total, hkv, torch.bfloat16, 80)
    q = (torch.randn(batch, hkv, hq // hkv, D, generator=g, device=DEV) + 0.3 * lean).reshape(batch, hq, D).to(torch.bfloat16)
    status = torch.zeros(1, **I32)
    out = ops.shared_prefix_attn(q, k, v, torch.tensor([0, batch], **I32), pptr, pidx, plast, ptr, idx, last, max_pages=4, status=status)
    assert int(status) == 0
    gq = hq // hkv
    for b in list(range(batch))[:: max(1, batch // 20)]:
        for h in range(hkv):
            kk, vv = (torch.cat([dense(x, pptr, pidx, 0, 60, h), dense(x, ptr, idx, b, own[b], h)]) for x in (k, v))
            ref, _, p = attend64(q[b, h * gq: (h + 1) * gq].double(), kk, vv, torch.ones(gq, kk.shape[0], dtype=torch.bool, device=DEV))
            assert ((out[b, h * gq: (h + 1) * gq].double() - ref).abs() <= tol_of(torch.bfloat16, p, vv, ref)).all(), (b, h)


def test_selection_flags_what_it_leaves_out_and_counts_every_slot():
    new, old, hq, hkv, block = [70, 0, 5, 130], [300, 900, 40, 1000], 8, 2, 32
    q, k, v, qo, tab, lens = make_prompt(new, old, hq, hkv, torch.bfloat16, seed=90)
    most = max((n + 15) // 16 for n in lens)
    meta = torch.stack([k.amin(2), k.amax(2)], 2).contiguous()
    slots = sum(new) // block + len(new)

    def call(qo=qo, tab=tab, max_pages=most, rows=None):
        status, count = torch.zeros(1, **I32), torch.full((slots, hkv), 99, **I32)
        pages = ops.quest_select_blocks(q, meta, qo, *tab, 128, max_pages=max_pages, query_block=block, block_npages=count,
                                        status=status)[0]
        return pages, count, int(status)

    def slots_of(b):
        first = int(qo[b]) // block + b
        return range(first, first + (new[b] + block - 1) // block)

    used = sorted(s for b in range(4) for s in slots_of(b))
    none = [s for s in range(slots) if s not in used]
    pages, count, status = call()
    assert status == 0 and none and (count[none] == 0).all() and (count[used] > 0).all() and (count <= pages.shape[2]).all()
    # a sequence that makes no sense: flagged, without lists; the others as before
    for b, last in ((0, 0), (3, 17)):
        wrong = tab[2].clone()
        wrong[b] = last
        got_pages, got, status = call(tab=(tab[0], tab[1], wrong))
        assert status == ops.FLAG_BAD_INDEX and (got[list(slots_of(b))] == 0).all()
        for s in used:
            if s not in slots_of(b):
                assert torch.equal(got[s], count[s])
                for h in range(hkv):
                    assert torch.equal(got_pages[s, h, : count[s, h]], pages[s, h, : count[s, h]])
    far = qo.clone()
    far[4] += 1                                                 # more rows than q has
    _, got, status = call(qo=far)
    assert status == ops.FLAG_BAD_INDEX and (got[list(slots_of(3))] == 0).all()
    # fewer pages than a sequence has: what is left out is flagged, and the lists stay in range
    got_pages, got, status = call(max_pages=most - 1)
    assert status == ops.FLAG_BAD_INDEX and (got <= got_pages.shape[2]).all()
    for s in used:
        for h in range(hkv):
            x = got_pages[s, h, : got[s, h]]
            assert (x[1:] > x[:-1]).all() and ((x >= 0) & (x < most - 1)).all()
    # a sequence without new tokens has no lists to leave anything out of
    assert call(max_pages=most)[2] == 0 and (lens[1] + 15) // 16 < most


@pytest.mark.parametrize("tokens, pages", [(3, (1 << 22) + 9), (40, (1 << 26) + 9)])
def test_a_list_shorter_than_its_place_at_far_positions(tokens, pages):
    """Positions beyond 2^26 and 2^30 (every page of the table is the same one): the places that a list leaves empty are no keys."""
    k, v, lean, g = pool(1, 1, torch.bfloat16, 95)
    q = torch.randn(tokens, 1, D, generator=g, device=DEV).to(torch.bfloat16)
    ptr, last = torch.tensor([0, pages], **I32), torch.tensor([16], **I32)
    idx = torch.zeros(pages, **I32)
    slots = tokens // 64 + 1
    lists, count = torch.zeros(slots, 1, 12, **I32), torch.ones(slots, 1, **I32)
    status = torch.zeros(1, **I32)
    out, lse = ops.prompt_attn(q, k, v, torch.tensor([0, tokens], **I32), ptr, idx, last, max_pages=pages, block_pages=lists,
                               block_npages=count, query_block=64, lse=True, status=status)
    assert int(status) == 0
    ref, ref_lse, p = attend64(q[:, 0].double(), k[0, 0].double(), v[0, 0].double(),
                               torch.ones(tokens, PAGE, dtype=torch.bool, device=DEV))
    assert ((out[:, 0].double() - ref).abs() <= tol_of(torch.bfloat16, p, v[0, 0].double(), ref)).all()
    assert ((lse[:, 0].double() - ref_lse).abs() <= 2.0 ** -18 + 2.0 ** -22 * ref_lse.abs()).all()


def test_more_new_tokens_than_the_sequence_has():
    """Queries before position 0 see nothing: zeros, whichever kernel takes them."""
    for new, old in (([5], [-3]), ([300], [-100])):
        lens = [new[0] + old[0]]
        ptr, idx, last = table(lens, 3)
        k, v, lean, g = pool(idx.numel(), 2, torch.float16, 96)
        q = torch.randn(new[0], 4, D, generator=g, device=DEV).half()
        qo = torch.tensor([0, new[0]], **I32)
        out, lse = ops.prompt_attn(q, k, v, qo, ptr, idx, last, max_pages=20, lse=True)
        check_prompt(q, k, v, qo, (ptr, idx, last), lens, out, lse)
        assert not out[: -old[0]].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [2, 40])
def test_many_small_weights_add_up(dtype, tokens):
    """One key of weight 1 and 2^18 of 2^-26.5 each, 2^-8.5 together: rounded to fp16 as they are they would all be zero."""
    n = 1 << 18
    k, v = (torch.zeros(2, 1, PAGE, D, dtype=dtype, device=DEV) for _ in range(2))
    k[0, 0, 0, 0] = 13.0
    v[:] = torch.randn(2, 1, 1, D, generator=torch.Generator(device=DEV).manual_seed(97), device=DEV).to(dtype)
    q = torch.zeros(tokens, 1, D, dtype=dtype, device=DEV)
    q[:, 0, 0] = 16.0
    idx = torch.ones(n // PAGE, **I32)
    idx[0] = 0
    tab = torch.tensor([0, n // PAGE], **I32), idx, torch.tensor([16], **I32)
    kk, vv = (x[idx.long(), 0].reshape(-1, D).double() for x in (k, v))
    keep = torch.ones(1, n, dtype=torch.bool, device=DEV)
    ref, _, p = attend64(q[:1, 0].double(), kk, vv, keep)
    tol = tol_of(dtype, p, vv, ref)
    assert ((ref - vv[:1]).abs() > 2 * tol).any()               # the small ones count
    out = ops.prompt_attn(q, k, v, torch.tensor([0, tokens], **I32), *tab, max_pages=n // PAGE, causal=False)
    assert ((out[:, 0].double() - ref).abs() <= tol).all()
    none = torch.zeros(tokens + 1, **I32), torch.zeros(0, **I32), torch.zeros(tokens, **I32)
    out = ops.shared_prefix_attn(q, k, v, torch.tensor([0, tokens], **I32), *tab, *none)
    assert ((out[:, 0].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chosen_pages_of_the_longest_history(dtype):
    """As many pages as the selection takes, a few hundred different ones: equal scores everywhere."""
    pages, new, hkv, block = 51200, 40, 2, 32
    k, v, lean, g = pool(300, hkv, dtype, 98)
    meta = torch.stack([k.amin(2), k.amax(2)], 2).contiguous()
    q = torch.randn(new, 4, D, generator=g, device=DEV).to(dtype)
    idx = torch.randint(0, 300, (pages,), generator=g, device=DEV, dtype=torch.int32)
    tab, qo = (torch.tensor([0, pages], **I32), idx, torch.tensor([16], **I32)), torch.tensor([0, new], **I32)
    for budget in (16, 5000, 700000):
        status = torch.zeros(1, **I32)
        got = ops.quest_select_blocks(q, meta, qo, *tab, budget, max_pages=pages, query_block=block, status=status)
        assert int(status) == 0
        assert exact_lists(q, meta, qo, tab, [pages * PAGE], budget, block, hkv, *got) == 2 * hkv


@pytest.mark.parametrize("scale", [1e-30, 1e-36, 1e-38])
def test_chosen_pages_of_queries_near_the_smallest_numbers(scale):
    q, k, v, qo, tab, lens = make_prompt([100], [3000], 4, 2, torch.bfloat16, seed=99)
    q = (q.double() * scale).to(torch.bfloat16)
    meta = ops.build_page_meta(k, *tab, max_pages=200)
    got = ops.quest_select_blocks(q, meta, qo, *tab, 500, max_pages=200, query_block=32)
    assert exact_lists(q, meta, qo, tab, lens, 500, 32, 2, *got) > 0
