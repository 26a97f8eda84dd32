"""Rotary positions with the ragged cache append, and INT4 slabs read back, against plain 64-bit implementations."""
import pytest
import torch

from twilight_b200.cache import PAGE, PagedKVCache, unpack_k4
from twilight_b200.kernel import ops

pytestmark = pytest.mark.gpu
DEV, D = "cuda", 128


def rotate64(x, pos, freqs, scale, inter):
    """x [T,H,128] in 64 bits, pos [T], freqs [R/2] -> rotated in 64 bits."""
    r = 2 * len(freqs)
    a = (pos.double()[:, None] * freqs.double().cpu())[:, None]
    c, s = a.cos() * scale, a.sin() * scale
    y = x.clone()
    u, v = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., : r // 2], x[..., r // 2: r])
    nu, nv = u * c - v * s, v * c + u * s
    if inter:
        y[..., 0:r:2], y[..., 1:r:2] = nu, nv
    else:
        y[..., : r // 2], y[..., r // 2: r] = nu, nv
    return y


def make(new, old, hq, hkv, dtype, seed=0, strided=True):
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, old)]
    indptr, indices, last, total = PagedKVCache.page_table([max(n, 1) for n in lens], DEV, seed + 1)
    last = torch.tensor([(n - 1) % PAGE + 1 if n else 1 for n in lens], dtype=torch.int32, device=DEV)
    pool = torch.randn(2, total, hkv, PAGE, D, generator=g).to(dtype)
    k, v = pool[0].to(DEV), pool[1].to(DEV)
    t = sum(new)
    proj = torch.randn(t, hq + 2 * hkv + 1, D, generator=g).to(dtype).to(DEV)
    parts = (proj[:, :hq], proj[:, hq: hq + hkv], proj[:, hq + hkv: hq + 2 * hkv])
    if not strided:
        parts = tuple(x.contiguous() for x in parts)
    qo = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return parts, k, v, (qo, indptr, indices, last), lens


CASES = [
    # new, old, hq, hkv, rotary, interleaved, dtype
    ([1], [0], 4, 1, 128, False, torch.bfloat16),
    ([1, 1, 1], [15, 16, 17], 8, 2, 128, False, torch.float16),
    ([1] * 40, list(range(40)), 3, 3, 64, True, torch.bfloat16),
    ([5, 0, 33, 16], [0, 7, 31, 16], 6, 2, 96, False, torch.float16),
    ([100, 1, 257], [3, 0, 250], 7, 1, 8, True, torch.bfloat16),
    ([700], [13], 32, 8, 128, True, torch.float16),
    ([31, 2, 16, 15, 17, 48], [1, 15, 0, 1, 15, 8], 5, 5, 32, False, torch.bfloat16),
    ([9, 20], [0, 30], 2, 2, 0, False, torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("positions", [None, torch.int32, torch.int64])
def test_rotates_writes_quantises_and_folds(case, positions):
    new, old, hq, hkv, rotary, inter, dtype = case
    (q, k, v), kp, vp, table, lens = make(new, old, hq, hkv, dtype)
    qo, indptr, indices, last = table
    scale = 1.25 if positions is torch.int32 else 1.0
    freqs, _ = ops.rope_frequencies(rotary, 500000.0, device=DEV) if rotary else (None, 1.0)
    slot = torch.cat([torch.arange(o, o + n) for n, o in zip(new, old)])
    pos = slot
    if positions is not None:
        pos = slot * 97 + 100003                                    # far ones, not the slots
    k0, v0 = kp.clone(), vp.clone()
    k4 = ops.quantize_k_pages(kp)
    k4_0 = k4.clone()
    meta = torch.stack([kp.amin(3 - 1), kp.amax(2)], 2).contiguous()
    meta0 = meta.clone()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.rope_append_kv(q, k, v, freqs, kp, vp, k4, meta, *table, interleaved=inter, attention_scale=scale,
                             positions=None if positions is None else pos.to(positions).to(DEV), status=status)
    assert int(status) == 0
    f64 = freqs.cpu() if rotary else torch.zeros(0, dtype=torch.float64)
    eps = torch.finfo(dtype).eps
    ids = torch.cat([indices.cpu()[int(indptr[b]) + torch.arange(o, o + n) // PAGE]
                     for b, (n, o) in enumerate(zip(new, old))]).long()

    def near(out, x):
        ref = rotate64(x.double().cpu(), pos, f64, scale, inter)
        # half a step of the type, and 32-bit sine, products and sum: below 2^-20 of the pair's length
        length = x.double().cpu().abs().amax(-1, keepdim=True) * 1.5 * scale
        # a value below the type's smallest normal number is rounded to its fixed step
        tiny = torch.finfo(dtype).smallest_normal * eps
        assert ((out.double().cpu() - ref).abs() <= eps / 2 * ref.abs() + length * 2.0 ** -20 + tiny).all()

    near(got, q)
    rows = kp.cpu()[ids, :, slot % PAGE]
    near(rows, k)
    assert torch.equal(vp.cpu()[ids, :, slot % PAGE], v.cpu())
    # everything else is as it was
    is_new = torch.zeros(kp.shape[0], PAGE, dtype=torch.bool)
    is_new[ids, slot % PAGE] = True
    keep = ~is_new[:, None].expand(-1, hkv, -1)
    assert torch.equal(kp.cpu()[keep], k0.cpu()[keep]) and torch.equal(vp.cpu()[keep], v0.cpu()[keep])
    # the slabs are those of the page quantiser on the rows now in the pages
    c, s, z = unpack_k4(k4.cpu())
    c1, s1, z1 = unpack_k4(ops.quantize_k_pages(kp).cpu())
    c0, s0, z0 = unpack_k4(k4_0.cpu())
    m = is_new[:, None].expand(-1, hkv, -1)
    for a, b, was in ((c, c1, c0), (s, s1, s0), (z, z1, z0)):
        assert torch.equal(a[m], b[m]) and torch.equal(a[~m], was[~m])
    # metadata: what the page held before where its first row is an old one, and its new rows
    want = meta0.cpu().float()
    for page in ids.unique().tolist():
        x = kp.cpu()[page][:, is_new[page]].float()
        lo, hi = x.amin(1), x.amax(1)
        if not is_new[page, 0]:
            lo, hi = torch.minimum(lo, want[page, :, 0]), torch.maximum(hi, want[page, :, 1])
        want[page, :, 0], want[page, :, 1] = lo, hi
    assert torch.equal(meta.cpu().float(), want)


def test_one_token_form_equals_append_kv_and_optional_parts():
    (q, k, v), kp, vp, table, lens = make([1] * 9, [0, 1, 15, 16, 30, 31, 32, 100, 7], 8, 4, torch.bfloat16)
    kp2, vp2 = kp.clone(), vp.clone()
    k4 = torch.zeros(kp.shape[0], 4, 1280, dtype=torch.uint8, device=DEV)
    meta = torch.zeros(kp.shape[0], 4, 2, D, dtype=kp.dtype, device=DEV)
    k4b, metab = k4.clone(), meta.clone()
    got = ops.rope_append_kv(q, k, v, None, kp, vp, k4, meta, *table)
    assert torch.equal(got, q)
    ops.append_kv(k.contiguous(), v.contiguous(), kp2, vp2, k4b, metab, *table[1:])
    for a, b in ((kp, kp2), (vp, vp2), (k4, k4b), (meta, metab)):
        assert torch.equal(a, b)
    freqs, _ = ops.rope_frequencies(128, device=DEV)
    kp3, vp3 = kp.clone(), vp.clone()
    ops.rope_append_kv(q, k, v, freqs, kp, vp, k4, meta, *table)
    out = q.clone()
    same = ops.rope_append_kv(out, k, v, freqs, kp3, vp3, None, None, *table, out=out)   # in place, pages only
    assert torch.equal(kp, kp3) and torch.equal(vp, vp3)
    assert torch.equal(same, ops.rope_append_kv(q, k, v, freqs, kp3, vp3, None, None, *table))


def test_bad_pages_and_lengths_are_flagged_and_skipped():
    (q, k, v), kp, vp, (qo, indptr, indices, last), _ = make([4, 20, 3], [0, 0, 40], 4, 2, torch.float16)
    k0, v0 = kp.clone(), vp.clone()
    bad = indices.clone()
    bad[int(indptr[1])] = 10 ** 6                          # the second sequence's first page
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    freqs, _ = ops.rope_frequencies(128, device=DEV)
    got = ops.rope_append_kv(q, k, v, freqs, kp, vp, None, None, qo, indptr, bad, last, status=status)
    assert int(status) == ops.FLAG_BAD_INDEX
    want = ops.rope_append_kv(q, k, v, freqs, k0.clone(), v0.clone(), None, None, qo, indptr, indices, last)
    assert torch.equal(got, want)                          # q is rotated all the same
    assert torch.equal(kp[int(indices[int(indptr[1])])], k0[int(indices[int(indptr[1])])])
    # more new tokens than the table says there are: that sequence is skipped
    short = last.clone()
    short[0] = 2
    status.zero_()
    kp4, vp4 = k0.clone(), v0.clone()
    ops.rope_append_kv(q, k, v, freqs, kp4, vp4, None, None, qo, indptr, indices, short, status=status)
    assert int(status) == ops.FLAG_BAD_INDEX
    assert torch.equal(kp4[int(indices[0])], k0[int(indices[0])])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_dequantised_values(dtype):
    g = torch.Generator().manual_seed(3)
    k = torch.randn(37, 3, PAGE, D, generator=g).to(dtype).to(DEV)
    k[5] = 0.5                                              # groups without a range
    k4 = ops.quantize_k_pages(k)
    codes, scale, zmin = unpack_k4(k4.cpu())
    want = (codes.unflatten(-1, (4, 32)).double() * scale.double()[..., None] + zmin.double()[..., None]).flatten(-2)
    got = ops.dequantize_k_pages(k4, dtype=dtype)
    eps = torch.finfo(dtype).eps
    tol = eps / 2 * want.abs() + 2.0 ** -22 * (15 * scale.abs() + zmin.abs()).double().amax() + \
        torch.finfo(dtype).smallest_normal * eps
    assert ((got.cpu().double() - want).abs() <= tol).all()
    ids = torch.tensor([36, 0, 5, 5], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.dequantize_k_pages(k4, ids, dtype=dtype), got[ids.long()])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    bad = ops.dequantize_k_pages(k4, torch.tensor([1, 37, -1], dtype=torch.int32, device=DEV), dtype=dtype, status=status)
    assert int(status) == ops.FLAG_BAD_INDEX and torch.equal(bad[0], got[1]) and not bad[1:].any()


def test_runs_under_graph_capture_and_on_a_side_stream():
    (q, k, v), kp, vp, table, _ = make([3, 40], [5, 0], 8, 2, torch.bfloat16)
    freqs, _ = ops.rope_frequencies(64, device=DEV)
    kw, vw = kp.clone(), vp.clone()
    want = ops.rope_append_kv(q, k, v, freqs, kw, vw, None, None, *table)
    out = torch.empty_like(want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.rope_append_kv(q, k, v, freqs, kp, vp, None, None, *table, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(kp, kw) and torch.equal(vp, vw)


@pytest.mark.parametrize("lead", [1, 16, 100, 161])
def test_rows_before_the_first_sequence_and_behind_the_last_are_left(lead):
    """Offsets that begin behind row 0: a part of a larger batch."""
    new, old = [4, 40, 1], [0, 3, 700]
    (q, k, v), kp, vp, (qo, *table), _ = make(new, old, 4, 2, torch.bfloat16, strided=False)
    freqs, _ = ops.rope_frequencies(128, device=DEV)
    k_want, v_want = kp.clone(), vp.clone()
    want = ops.rope_append_kv(q, k, v, freqs, k_want, v_want, None, None, qo, *table)
    wide = [torch.nn.functional.pad(x, (0, 0, 0, 0, lead, 7), value=3.0) for x in (q, k, v)]
    out = torch.full_like(wide[0], 5.0)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope_append_kv(*wide, freqs, kp, vp, None, None, qo + lead, *table, out=out, status=status)
    t = q.shape[0]
    assert int(status) == 0 and torch.equal(out[lead: lead + t], want)
    assert torch.equal(kp, k_want) and torch.equal(vp, v_want)
    assert (out[:lead] == 5).all() and (out[lead + t:] == 5).all()


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("pad", [0, 4])
def test_in_place(case, pad):
    """out as q itself: rows of a fused projection; with `pad` more elements a head they start anywhere in a 32-byte sector."""
    new, old, hq, hkv, rotary, inter, dtype = case
    (q, k, v), kp, vp, table, lens = make(new, old, hq, hkv, dtype)
    freqs, scale = ops.rope_frequencies(rotary, device=DEV) if rotary else (None, 1.0)
    kw = dict(interleaved=inter, attention_scale=scale)
    want = ops.rope_append_kv(q, k, v, freqs, kp.clone(), vp.clone(), None, None, *table, **kw)
    wide = torch.zeros(q.shape[0], hq + 1, D + pad, dtype=dtype, device=DEV)
    mine = wide[:, :hq, :D]
    mine.copy_(q)
    got = ops.rope_append_kv(mine, k, v, freqs, kp, vp, None, None, *table, out=mine, **kw)
    assert got.data_ptr() == mine.data_ptr() and torch.equal(got, want)
    assert not wide[:, hq].any() and not wide[..., D:].any()


def test_strides_of_one_token_and_of_one_head_are_not_read():
    for new, hq, hkv in (([1], 4, 2), ([9, 3], 1, 1), ([1], 1, 1)):
        (q, k, v), kp, vp, table, lens = make(new, [20] * len(new), hq, hkv, torch.bfloat16)
        freqs, _ = ops.rope_frequencies(device=DEV)
        t = sum(new)

        def odd(x):
            x = x.contiguous()
            return torch.as_strided(x, x.shape, (13 if t == 1 else x.stride(0), 7 if x.shape[1] == 1 else D, 1))

        pools = [x.clone() for x in (kp, vp)]
        want = ops.rope_append_kv(q, k, v, freqs, *pools, None, None, *table)
        out = odd(torch.zeros(t, hq, D, dtype=q.dtype, device=DEV))
        got = ops.rope_append_kv(odd(q), odd(k), odd(v), freqs, kp, vp, None, None, *table, out=out)
        assert torch.equal(got, want) and torch.equal(kp, pools[0]) and torch.equal(vp, pools[1])
