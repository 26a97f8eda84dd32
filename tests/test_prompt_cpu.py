"""Host side of the prompt operators: frequencies, argument checks and status codes (no kernel is launched)."""
import math

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
    (dict(k=torch.zeros(4, 1, 128, dtype=torch.float16)), "k has 1 heads"),
    (dict(v=torch.zeros(5, 2, 128, dtype=torch.float16)), "same tokens"),
    (dict(k=torch.zeros(4, 2, 128, dtype=torch.bfloat16)), "same tokens and type"),
    (dict(q=torch.zeros(4, 3, 128, dtype=torch.float16)), "multiple of KV heads"),
    (dict(kmeta=torch.zeros(3, 2, 2, 128, dtype=torch.bfloat16)), "kmeta is"),
    (dict(v_pages=torch.zeros(4, 2, 16, 128, dtype=torch.float16)), "same pages"),
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
