"""Host side of the prompt operators: frequencies, argument checks and status codes (no kernel is launched)."""
import math
import re
from pathlib import Path

import pytest
import torch

from twilight_b200 import _lib
from twilight_b200.kernel import ops


def test_rope_frequencies_of_the_known_scalings():
    f, s = ops.rope_frequencies(128, 10000.0, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64)
    assert s == 1.0 and torch.allclose(f, want, rtol=1e-14) and f.dtype == torch.float64
    lin, s = ops.rope_frequencies(64, 5e5, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert s == 1.0 and torch.allclose(lin, ops.rope_frequencies(64, 5e5, device="cpu")[0] / 4, rtol=1e-14)
    # llama3: wavelengths below original/high unchanged, above original/low divided by the factor, a ramp between
    sc = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    base = ops.rope_frequencies(128, 5e5, device="cpu")[0]
    l3, s = ops.rope_frequencies(128, 5e5, scaling=sc, device="cpu")
    wave = 2 * math.pi / base
    assert s == 1.0 and torch.allclose(l3[wave < 8192 / 4], base[wave < 8192 / 4], rtol=1e-14)
    assert torch.allclose(l3[wave > 8192], base[wave > 8192] / 8, rtol=1e-14)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    smooth = (8192 / wave[mid] - 1) / 3
    assert mid.any() and torch.allclose(l3[mid], (1 - smooth) * base[mid] / 8 + smooth * base[mid], rtol=1e-12)
    # yarn: fast pairs kept, slow ones divided, cos and sin scaled
    sc = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 8192}
    y, s = ops.rope_frequencies(128, 5e5, scaling=sc, device="cpu")
    assert math.isclose(s, 0.1 * math.log(16) + 1) and y[0] == base[0] and math.isclose(y[-1], base[-1] / 16)
    assert ((y <= base) & (y >= base / 16)).all()
    assert ops.rope_frequencies(128, 5e5, scaling={**sc, "attention_factor": 1.5}, device="cpu")[1] == 1.5
    # dynamic: unchanged up to the original length, a larger base beyond it
    sc = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    assert torch.equal(ops.rope_frequencies(128, 1e4, scaling=sc, seq_len=4000, device="cpu")[0],
                       ops.rope_frequencies(128, 1e4, device="cpu")[0])
    d, _ = ops.rope_frequencies(128, 1e4, scaling=sc, seq_len=16384, device="cpu")
    b = 1e4 * (2 * 16384 / 4096 - 1) ** (128 / 126)
    assert math.isclose(d[5].item(), b ** (-10 / 128), rel_tol=1e-12)
    with pytest.raises(_lib.TwilightError, match="rope_type"):
        ops.rope_frequencies(128, scaling={"rope_type": "nope"}, device="cpu")
    for bad in (0, 12, 136):
        with pytest.raises(_lib.TwilightError, match="rotary_dim"):
            ops.rope_frequencies(bad, device="cpu")


def test_rope_frequencies_refuses_what_it_would_get_wrong():
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    freq = lambda sc, dim=128, base=1e4: ops.rope_frequencies(dim, base, scaling=sc, device="cpu")
    for sc, said in (({**yarn, "mscale": 1.0}, "mscale"), ({**yarn, "mscale_all_dim": 0.7}, "mscale_all_dim"),
                     ({"rope_type": "yarn", "factor": 4.0}, "original_max"), ({"rope_type": "linear"}, "factor"),
                     ({"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192}, "low_freq"),
                     ({"rope_type": "dynamic", "factor": 2.0, "alpha": 8.0}, "lacks"),
                     ({"rope_type": "linear", "factor": 2.0, "short_factor": [1.0]}, "short_factor"),
                     ({**yarn, "rope_theta": 5e5}, "rope_theta"), ({**yarn, "partial_rotary_factor": 0.5}, "partial")):
        with pytest.raises(_lib.TwilightError, match=said):
            freq(sc)
    # what does not matter, or says what the arguments say, is taken
    assert torch.equal(freq({**yarn, "rope_theta": 10000.0, "partial_rotary_factor": 1.0, "beta_fast": None})[0], freq(yarn)[0])
    f, s = freq({**yarn, "attention_factor": 1.2, "mscale": 1.0, "mscale_all_dim": 1.0})
    assert s == 1.2 and torch.equal(f, freq(yarn)[0])
    # fractional ends of the ramp
    f, _ = freq({**yarn, "truncate": False})
    base = freq(None)[0]
    ends = [128 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(1e4)) for t in (32.0, 1.0)]
    ramp = ((torch.arange(64, dtype=torch.float64) - ends[0]) / (ends[1] - ends[0])).clamp(0, 1)
    assert torch.allclose(f, base * (1 - ramp) + base / 4 * ramp, rtol=1e-12) and not torch.equal(f, freq(yarn)[0])


def _append_args(t=4, hq=4, hkv=2, dtype=torch.float16):
    q, k, v = (torch.zeros(t, h, 128, dtype=dtype) for h in (hq, hkv, hkv))
    kp, vp = (torch.zeros(3, hkv, 16, 128, dtype=dtype) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=q, k=k, v=v, freqs=torch.ones(64, dtype=torch.float64), k_pages=kp, v_pages=vp,
                k4_pages=torch.zeros(3, hkv, 1280, dtype=torch.uint8), kmeta=torch.zeros(3, hkv, 2, 128, dtype=dtype),
                qo_indptr=i32([0, 1, t]), kv_indptr=i32([0, 1, 3]), kv_indices=i32([0, 1, 2]),
                kv_last_page_len=i32([3, 4]))


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(4, 4, 64, dtype=torch.float16)), "q must be"),
    (dict(k=torch.zeros(4, 1, 128, dtype=torch.float16)), "cache's 2 heads"),
    (dict(v=torch.zeros(5, 2, 128, dtype=torch.float16)), "q's tokens"),
    (dict(k=torch.zeros(4, 2, 128, dtype=torch.bfloat16)), "tokens and type"),
    (dict(q=torch.zeros(4, 3, 128, dtype=torch.float16)), "multiple of KV heads"),
    (dict(kmeta=torch.zeros(3, 2, 2, 128, dtype=torch.bfloat16)), "kmeta is"),
    (dict(v_pages=torch.zeros(4, 2, 16, 128, dtype=torch.float16)), "pages and heads of k_pages"),
    (dict(k4_pages=torch.zeros(3, 2, 1024, dtype=torch.uint8)), "k4_pages"),
    (dict(kv_last_page_len=torch.zeros(3, dtype=torch.int32)), "kv_last_page_len must have 2"),
    (dict(kv_indices=torch.zeros(3, dtype=torch.int64)), "kv_indices must be"),
    (dict(freqs=torch.ones(64)), "float64"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), "positions"),
    (dict(out=torch.zeros(4, 4, 128)), "out must have"),
    ({}, "CUDA tensors only"),
])
def test_rope_append_refuses(change, match):
    with pytest.raises(_lib.TwilightError, match=match):
        ops.rope_append_kv(**{**_append_args(), **change})


def test_dequantize_refuses():
    k4 = torch.zeros(3, 2, 1280, dtype=torch.uint8)
    with pytest.raises(_lib.TwilightError, match="CUDA tensor"):
        ops.dequantize_k_pages(k4, dtype=torch.float16)
    lib = _lib.load()
    assert lib.twl_dequantize_k_pages(None, None, 1, None, 0, 1, 1, None, None) == -1
    assert lib.twl_dequantize_k_pages(256, None, 4, 256, 0, 1, 3, None, None) == -1    # more pages than there are
    assert lib.twl_dequantize_k_pages(256, None, 1, 256, 7, 1, 3, None, None) == -3
    assert lib.twl_dequantize_k_pages(256, None, 1, 264, 0, 1, 3, None, None) == -2


def _rope_c(**kw):
    a = dict(q=256, k=256, v=256, dtype=0, s=(512, 128, 256, 128, 256, 128), out=256, os=(512, 128), pos=None, p64=0,
             freqs=256, rot=128, inter=0, scale=1.0, kp=256, vp=256, k4=None, meta=None, qo=256, ip=256, idx=256, ll=256,
             t=4, b=2, hq=4, hkv=2, pages=3)
    a.update(kw)
    return _lib.load().twl_rope_append_kv(a["q"], a["k"], a["v"], a["dtype"], *a["s"], a["out"], *a["os"], a["pos"],
                                          a["p64"], a["freqs"], a["rot"], a["inter"], a["scale"], a["kp"], a["vp"],
                                          a["k4"], a["meta"], a["qo"], a["ip"], a["idx"], a["ll"], a["t"], a["b"],
                                          a["hq"], a["hkv"], a["pages"], None, None)


def test_rope_append_status_codes():
    assert _rope_c(q=None) == _rope_c(t=0) == _rope_c(hq=3) == _rope_c(freqs=None) == _rope_c(rot=-8) == -1
    assert _rope_c(rot=12) == _rope_c(rot=8) == _rope_c(rot=136) == _rope_c(dtype=5) == -3
    assert _rope_c(q=260) == _rope_c(s=(510, 128, 256, 128, 256, 128)) == _rope_c(kp=264) == _rope_c(meta=8) == -2
    assert _rope_c(hq=65536, hkv=65536) == -5


def _prompt_args(t=40, hq=4, hkv=2, dtype=torch.bfloat16):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros(t, hq, 128, dtype=dtype), k_pages=torch.zeros(3, hkv, 16, 128, dtype=dtype),
                v_pages=torch.zeros(3, hkv, 16, 128, dtype=dtype), qo_indptr=i32([0, 1, t]), kv_indptr=i32([0, 1, 3]),
                kv_indices=i32([0, 1, 2]), kv_last_page_len=i32([3, 4]), max_pages=2)


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(40, 4, 64, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(4, 40, 128, dtype=torch.bfloat16).transpose(0, 1)), "heads of a token contiguous"),
    (dict(q=torch.zeros(40, 3, 128, dtype=torch.bfloat16)), "multiple of KV heads"),
    (dict(v_pages=torch.zeros(3, 2, 16, 128)), "v_pages is"),
    (dict(k_pages=torch.zeros(3, 2, 128, 16, dtype=torch.bfloat16)), "k_pages must be"),
    (dict(kv_indptr=torch.zeros(5, dtype=torch.int32)), "kv_indptr must have 3"),
    (dict(qo_indptr=torch.zeros(3, dtype=torch.int64)), "qo_indptr must be"),
    (dict(out=torch.zeros(40, 4, 128)), "out must be"),
    (dict(lse=torch.zeros(40, 3)), "lse must be"),
    (dict(block_pages=torch.zeros(2, 2, 4, dtype=torch.int32)), "go together"),
    (dict(block_pages=torch.zeros(1, 2, 4, dtype=torch.int32), block_npages=torch.zeros(2, 2, dtype=torch.int32)),
     "block_pages must be"),
    ({}, "CUDA tensors only"),
])
def test_prompt_attn_refuses(change, match):
    with pytest.raises(_lib.TwilightError, match=match):
        ops.prompt_attn(**{**_prompt_args(), **change})


@pytest.mark.parametrize("change, match", [
    (dict(token_budget=0), "must be positive"),
    (dict(query_block=40), "multiple of 16"),
    (dict(kmeta=torch.zeros(3, 2, 2, 128)), "kmeta is"),
    (dict(pooled=torch.zeros(2, 2, 128)), "pooled must be"),
    (dict(block_pages=torch.zeros(2, 2, 1, dtype=torch.int32)), "at least 2"),
    ({}, "CUDA tensors only"),
])
def test_quest_select_blocks_refuses(change, match):
    a = _prompt_args()
    a = {**{k: v for k, v in a.items() if k not in ("k_pages", "v_pages")}, "token_budget": 64, "query_block": 64,
         "kmeta": torch.zeros(3, 2, 2, 128, dtype=torch.bfloat16), **change}
    if "CUDA" not in match and "positive" not in match and "multiple of 16" not in match and "kmeta" not in match:
        real, ops._cuda = ops._cuda, lambda t: None      # past the device check, to the scratch buffers' own
        try:
            with pytest.raises(_lib.TwilightError, match=match):
                ops.quest_select_blocks(**a)
        finally:
            ops._cuda = real
        return
    with pytest.raises(_lib.TwilightError, match=match):
        ops.quest_select_blocks(**a)


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(3, 4, 2, 128, dtype=torch.bfloat16)), "q_len must be 1"),
    (dict(group_indptr=torch.zeros(0, dtype=torch.int32), prefix_indptr=torch.zeros(0, dtype=torch.int32)), "at least two entries"),
    (dict(prefix_last_page_len=torch.zeros(2, dtype=torch.int32)), "prefix_last_page_len must have 1"),
    (dict(kv_indices=torch.zeros(2)), "kv_indices must be"),
    (dict(workspace=torch.zeros(4)), "CUDA tensors only"),
])
def test_shared_prefix_refuses(change, match):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pools = torch.zeros(2, 3, 2, 16, 128, dtype=torch.bfloat16)
    a = dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16), k_pages=pools[0], v_pages=pools[1], group_indptr=i32([0, 3]),
             prefix_indptr=i32([0, 1]), prefix_indices=i32([0]), prefix_last_page_len=i32([16]),
             kv_indptr=i32([0, 1, 1, 2]), kv_indices=i32([1, 2]), kv_last_page_len=i32([1, 0, 2]))
    with pytest.raises(_lib.TwilightError, match=match):
        ops.shared_prefix_attn(**{**a, **change})


def test_attention_status_codes():
    lib = _lib.load()

    def prompt(**kw):
        a = dict(q=256, dtype=1, ts=512, k=256, v=256, qo=256, ip=256, idx=256, ll=256, t=4, b=2, hq=4, hkv=2, pages=3, mp=2,
                 causal=1, bp=None, bn=None, mk=0, qb=0, scale=0.1, out=256, lse=None, ws=256, wb=1 << 40)
        a.update(kw)
        return lib.twl_prompt_attn(*a.values(), None, None)

    assert prompt(q=None) == prompt(out=None) == prompt(hq=3) == prompt(mp=0) == prompt(bp=256) == prompt(scale=0.0) == -1
    assert prompt(scale=float("nan")) == prompt(bp=256, bn=256, mk=0, qb=64) == -1
    assert prompt(dtype=2) == prompt(hq=129 * 2) == prompt(bp=256, bn=256, mk=2, qb=40) == -3
    assert prompt(q=264) == prompt(ts=516) == prompt(k=264) == prompt(out=8) == -2
    assert prompt(ws=None) == prompt(wb=64) == prompt(ws=257) == -6
    assert prompt(pages=1 << 30) == -5
    need = lib.twl_prompt_attn_workspace_bytes(4, 2, 4, 2, 2, 0)
    assert 0 < need < 1 << 20 and lib.twl_prompt_attn_workspace_bytes(4, 2, 3, 2, 2, 0) == 0
    assert lib.twl_prompt_attn_workspace_bytes(32768, 1, 32, 8, 2048, 64) < 200 << 20
    assert lib.twl_shared_prefix_workspace_bytes(4, 0, 4, 2, 2) == 0
    assert lib.twl_shared_prefix_workspace_bytes(64, 1, 32, 8, 2048) < 200 << 20
    assert lib.twl_shared_prefix_attn(None, 1, 512, 256, 256, 256, 256, 256, 256, 256, 256, 256, 4, 1, 4, 2, 3, 2, 0.1, 256,
                                      None, 256, 1 << 40, None, None) == -1
    select = lambda **kw: lib.twl_quest_select_blocks(*{**dict(  # noqa: E731
        q=256, dtype=1, ts=512, meta=256, qo=256, ip=256, idx=256, ll=256, t=4, b=2, hq=4, hkv=2, pages=3, budget=64, qb=64,
        mp=2, pooled=256, scores=256, bp=256, bn=256, mk=2), **kw}.values(), None, None)
    assert select(budget=0) == select(pooled=None) == select(hq=5) == -1
    assert select(qb=24) == select(dtype=9) == -3 and select(ts=510) == -2 and select(mp=60000) == -5


def test_kernels_wait_before_they_read():
    """What an earlier kernel of the stream wrote is visible after griddepcontrol.wait only: in every kernel of the prompt
    operators that wait comes before the first read of memory."""
    csrc = Path(_lib.__file__).resolve().parent / "csrc"
    found = []
    for name in ("rope.cu", "prompt.cu", "prompt_tile.cu", "select.cu"):
        for kernel in re.finditer(r"__global__ void .*?\b(\w+_kernel)\(.*?\n}\n", (csrc / name).read_text(), re.S):
            if name == "select.cu" and "query_blocks" not in kernel.group(1):
                continue
            found.append(kernel.group(1))
            before = kernel.group(0)[: kernel.group(0).index("pdl_wait();")]
            assert not re.search(r"\bp\.\w+(\[|->)|__ld|ldg|load_|look_up|tma_|query_block", before.split("{", 1)[1]), found[-1]
    assert len(found) == 9, found


def planned_partials(own, sizes, prefix, hq, hkv):
    """Partial rows that the plan kernel hands out for shared_prefix_attn (csrc/prompt.cu) on a GPU of 148 SMs: lengths in pages."""
    g, sms, n = hq // hkv, 148, len(own)
    row_tile = 8 if g <= 8 and n * g > 16 else 16
    segs = [(1, x) for x in own] + list(zip(sizes, prefix))
    few = [s for s in segs if s[0] * g <= row_tile]
    tile = [(-(-t // (2 * (128 // g))) * hkv, t, pages) for t, pages in segs if t * g > row_tile]
    per = max(4, -(-sum(hkv * p for t, p in few if t) // (sms * (8 if row_tile == 8 else 7))))
    rows = sum(t * hq * (-(-p // per) + 1) for t, p in few)
    tiles, work = sum(x[0] for x in tile), sum(x[0] * x[2] for x in tile)
    share, tc = -(-work // sms), 0
    if tiles < sms:
        tc = (max(-(-work // (sms - tiles // 2)), 32) + 7) & ~7
        for _ in range(3):
            cut = [max(1, -(-p // tc)) for _, _, p in tile]
            items = sum(x[0] * c for x, c in zip(tile, cut))
            longest = max([0] + [-(-x[2] // c) for x, c in zip(tile, cut)])
            if items <= sms:
                break
            tc = (tc * items // sms + 8) & ~7
        if share * 5 < longest * 4 and share > 24 * 8:
            tc = 0
    if tc == 0:
        tc = (max((share + 2) // 3, 128) + 7) & ~7
    return rows + sum(max(1, -(-p // tc)) * t * hq for _, t, p in tile)


@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (32, 8), (9, 1), (16, 1), (17, 1), (32, 1), (33, 1), (48, 1), (96, 2), (64, 1), (128, 1)])
def test_workspace_of_a_shared_prefix_holds_its_partial_results(heads):
    lib, (hq, hkv) = _lib.load(), heads
    shapes = [([4] * n, [n], [4]) for n in (1, 2, 3, 20, 64)] + [([32] * 1000, [1000], [32]), ([1] * 2000, [700, 1300], [32, 1])]
    r = torch.Generator().manual_seed(hq)
    for _ in range(60):
        sizes = [int(torch.randint(0, 70, (1,), generator=r)) for _ in range(int(torch.randint(1, 5, (1,), generator=r)))]
        top = (1, 4, 32, 40, 300, 3000)[int(torch.randint(6, (1,), generator=r))]
        if sum(sizes):
            shapes.append((torch.randint(0, top + 1, (sum(sizes),), generator=r).tolist(), sizes,
                           torch.randint(0, top + 1, (len(sizes),), generator=r).tolist()))
    for own, sizes, prefix in shapes:
        most = max(1, max(own + prefix))
        size = lib.twl_shared_prefix_workspace_bytes(len(own), len(sizes), hq, hkv, most)
        # a partial row is 520 bytes; a segment 56, an item of the tile list (888 and more of them) 16, the header 256
        room = (size - 256 - 56 * (len(own) + len(sizes)) - 16 * 888) // 520
        assert planned_partials(own, sizes, prefix, hq, hkv) <= room, (len(own), sizes, most)


def test_rows_that_may_be_rotated_in_place_are_not_read_as_read_only():
    """rope_append_kv's out may be q itself; ld.global.nc is undefined for memory that the kernel writes."""
    text = (Path(_lib.__file__).resolve().parent / "csrc" / "rope.cu").read_text()
    kernel = text[text.index("rope_append_kernel("): text.index("struct DequantParams")]
    queries = kernel[kernel.index("static_cast<const T*>(p.q)"):]
    assert "p.q)" not in kernel[: -len(queries)] and not re.search(r"load_row16|ldg", queries)
    load_q = text[text.index("load_q16("): text.index("store_row16(")]
    assert "ld.global" in load_q and ".nc" not in load_q and "ldg" not in load_q


def test_workspace_sizes_are_those_of_the_device_of_the_call(monkeypatch):
    """A process with GPUs of different SM counts: a size asked for one is not given for the other."""
    sms, current = {0: 100, 1: 148}, [0]

    class Device:
        def __init__(self, index):
            self.index, self.before = index, current[0]

        def __enter__(self):
            current[0] = self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        twl_prompt_attn_workspace_bytes = staticmethod(lambda *a: sms[current[0]] * a[0])
        twl_shared_prefix_workspace_bytes = staticmethod(lambda *a: sms[current[0]] * a[0])

    monkeypatch.setattr(_lib, "load", lambda: Library)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    for size, args in ((ops.prompt_attn_workspace_bytes, (999983, 1, 8, 2, 4)),
                       (ops.shared_prefix_workspace_bytes, (999983, 1, 8, 2, 4))):
        for _ in range(2):
            for current[0] in (0, 1):
                assert size(*args) == sms[current[0]] * 999983
        current[0] = 0
        assert size(*args, device="cuda:1") == 148 * 999983 and size(*args, device="cuda:0") == 100 * 999983
        assert size(*args, device="cuda") == 100 * 999983 and current[0] == 0
    ops._workspace_bytes.cache_clear()
