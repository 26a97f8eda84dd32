"""Operator API of the Select-then-Prune decode path.

``top_p_fp32_return_mask`` / ``top_p_fp16_return_mask`` keep the names, arguments and result of
the reference's ``twilight.kernel`` (twilight/kernel/cuda/sampling.py:118-133).  The other
operators are the index-list forms the decode step is built from.  Every operator launches
hand-written sm_100a kernels through the C ABI on the current CUDA stream; none of them has a
PyTorch or CPU fallback.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple, Union

import torch

from .. import _lib

PAGE = 16
HEAD_DIM = 128
K4_SLAB_BYTES = 1280

FLAG_ITER_CAP, FLAG_BAD_INDEX, FLAG_WAIT_LIMIT = 1, 2, 4
_SM_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_INT32 = torch.int32


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float16:
        return 0
    if t.dtype == torch.bfloat16:
        return 1
    raise _lib.TwilightError(f"unsupported dtype {t.dtype}: the kernels take float16 or bfloat16")


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(device) -> int:
    # the raw handle (a Stream object costs 2 us a call on the host, what a small operator has to spare)
    index = device.index if device.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(index)


def _same_device(dev: torch.device, **tensors: Optional[torch.Tensor]) -> None:
    """Every tensor that crosses the C ABI in one call must live on the device the kernels run on."""
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise _lib.TwilightError(f"{name} is on {t.device}, the call runs on {dev}")


def _on(t: torch.Tensor, **others: Optional[torch.Tensor]):
    """Context in which ``t``'s device is the current CUDA device, as the reference's operators do
    with ``with probs.device`` (twilight/kernel/cuda/sampling.py:68).  The library launches on the
    current device, so a tensor on cuda:1 while cuda:0 is current (Hugging Face ``device_map="auto"``,
    benchmark/LongBench/pred.py:272-274) needs this guard; ``others`` are checked to be on that
    device too."""
    if not t.is_cuda:
        raise _lib.TwilightError("the operators take CUDA tensors only (there is no CPU path)")
    _same_device(t.device, **others)
    return torch.cuda.device(t.device)


def _cuda_contig(t: torch.Tensor, name: str) -> None:
    # same checks as CHECK_INPUT in csrc/src/pytorch_extension_utils.h:220-233
    if not t.is_cuda:
        raise _lib.TwilightError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise _lib.TwilightError(f"{name} must be contiguous")


def _q3(q: torch.Tensor) -> torch.Tensor:
    """Accepts q as [B,H,D] or the reference's [B,H,1,D]."""
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise _lib.TwilightError("decode step only: q_len must be 1")
        q = q[:, :, 0, :]
    if q.dim() != 3 or q.shape[-1] != HEAD_DIM:
        raise _lib.TwilightError(f"q must be [B,H,{HEAD_DIM}]")
    _cuda_contig(q, "q")
    return q


# ---------------------------------------------------------------------------------------------
# reference-compatible mask operators
# ---------------------------------------------------------------------------------------------
def _top_p_return_mask(probs: torch.Tensor, arr: Optional[torch.Tensor], val: float, half: bool
                       ) -> torch.Tensor:
    _cuda_contig(probs, "probs")
    if probs.dim() != 4:
        raise _lib.TwilightError("probs must be a 4D tensor")  # CHECK_DIM(4, probs)
    lib = _lib.load()
    b, h, _, d = probs.shape
    if arr is not None:
        arr = arr.to(device=probs.device, dtype=torch.float32).contiguous()
        if arr.numel() != b * h:
            raise _lib.TwilightError("top_p tensor must have batch*num_heads elements")
    with _on(probs):
        mask = torch.zeros_like(probs, dtype=torch.bool)
        if half:
            st = lib.twl_top_p_return_mask_f16(probs.data_ptr(), _dtype_code(probs), mask.data_ptr(),
                                               _p(arr), val, b * h, d, None, _stream(probs.device))
        else:
            if probs.dtype != torch.float32:
                raise _lib.TwilightError("top_p_fp32_return_mask takes float32 probabilities")
            st = lib.twl_top_p_return_mask_f32(probs.data_ptr(), mask.data_ptr(), _p(arr), val,
                                               b * h, d, None, _stream(probs.device))
    _lib.check(st, "top_p_return_mask")
    return mask


# The reference registers its two mask operators as torch custom ops without mutated arguments
# (``flashinfer::top_p_fp{16,32}_return_mask``, twilight/kernel/cuda/sampling.py:62-100), which is
# what lets them sit inside traced or compiled graphs.  Same here, under this library's namespace:
# ``torch.ops.twilight_b200.top_p_fp32_return_mask(probs, maybe_top_p_arr, top_p_val)``, with a
# fake-tensor rule.  Registered through ``torch.library.Library`` (a schema without aliased or
# mutated arguments says the same as ``mutates_args=()``): its dispatch costs about 3 us a call on
# the host against about 12 us for the ``custom_op`` decorator, which matters for small rows.
_TORCH_LIB = torch.library.Library("twilight_b200", "DEF")
_SCHEMA = "(Tensor probs, Tensor? maybe_top_p_arr, float top_p_val) -> Tensor"


def _op_top_p_fp32(probs: torch.Tensor, maybe_top_p_arr: Optional[torch.Tensor], top_p_val: float
                   ) -> torch.Tensor:
    return _top_p_return_mask(probs, maybe_top_p_arr, top_p_val, half=False)


def _op_top_p_fp16(probs: torch.Tensor, maybe_top_p_arr: Optional[torch.Tensor], top_p_val: float
                   ) -> torch.Tensor:
    return _top_p_return_mask(probs, maybe_top_p_arr, top_p_val, half=True)


def _fake_top_p_mask(probs, maybe_top_p_arr, top_p_val):
    return torch.empty_like(probs, dtype=torch.bool)


for _name, _impl in (("top_p_fp32_return_mask", _op_top_p_fp32), ("top_p_fp16_return_mask", _op_top_p_fp16)):
    _TORCH_LIB.define(_name + _SCHEMA)
    # every backend goes to the same function: it refuses anything that is not a CUDA tensor itself
    _TORCH_LIB.impl(_name, _impl, "CompositeExplicitAutograd")
    torch.library.register_fake("twilight_b200::" + _name, _fake_top_p_mask, lib=_TORCH_LIB)


def _to_tensor_scalar_tuple(x):
    # twilight/kernel/cuda/sampling.py:111-115
    return (x, 0.0) if isinstance(x, torch.Tensor) else (None, float(x))


def top_p_fp32_return_mask(probs: torch.Tensor, top_p: Union[torch.Tensor, float]) -> torch.Tensor:
    """probs ``[B,H,1,L]`` fp32 -> bool mask of the tokens the top-p search keeps
    (twilight/kernel/cuda/sampling.py:127-133, csrc/src/sampling.cu:45-63)."""
    return torch.ops.twilight_b200.top_p_fp32_return_mask(probs, *_to_tensor_scalar_tuple(top_p))


def top_p_fp16_return_mask(probs: torch.Tensor, top_p: Union[torch.Tensor, float]) -> torch.Tensor:
    """fp16/bf16 form (twilight/kernel/cuda/sampling.py:118-124, csrc/src/sampling.cu:22-43)."""
    return torch.ops.twilight_b200.top_p_fp16_return_mask(probs, *_to_tensor_scalar_tuple(top_p))


def _launch(name: str, on: torch.Tensor, *args, **same_device: Optional[torch.Tensor]) -> None:
    """Calls entry point ``twl_<name>`` with ``on``'s device current (the library launches on the
    current device); the keyword tensors are checked to live on that device.  Raises
    :class:`TwilightError` on a non-zero status."""
    lib = _lib.load()
    with _on(on, **same_device):
        st = getattr(lib, "twl_" + name)(*args)
    _lib.check(st, name)


def _launch_small(name: str, index: int, tensors, args) -> None:
    """:func:`_launch` for operators that can take less than ten microseconds on the GPU, where what the host does
    between two calls is what counts: ``tensors`` (name, tensor, name, tensor ..) are compared by device index, and no
    context is entered when the device is the current one."""
    for t in tensors[1::2]:
        if t is not None and t.get_device() != index:
            _same_device(torch.device("cuda", index), **dict(zip(tensors[::2], tensors[1::2])))
    fn = getattr(_lib.load(), "twl_" + name)
    if torch._C._cuda_getDevice() == index:
        st = fn(*args)
    else:
        with torch.cuda.device(index):
            st = fn(*args)
    if st != 0:
        _lib.check(st, name)


# ---------------------------------------------------------------------------------------------
# index-list operators
# ---------------------------------------------------------------------------------------------
def quest_page_scores(q, kmeta, kv_indptr, kv_indices, *, max_pages: int, page_scores=None, status=None
                      ) -> torch.Tensor:
    """Quest's per-page upper bounds ``sum_d max(q_d*kmax_d, q_d*kmin_d)`` from the stored page
    metadata, fp32 ``[B,H,max_pages]`` (twilight/pyimpl/quest.py:37-84)."""
    q = _q3(q)
    b, hq, _ = q.shape
    if page_scores is None:
        page_scores = torch.empty(b, hq, max_pages, dtype=torch.float32, device=q.device)
    _launch("quest_page_scores", q, q.data_ptr(), _dtype_code(q), kmeta.data_ptr(), kv_indptr.data_ptr(),
            kv_indices.data_ptr(), b, hq, kmeta.shape[1], kmeta.shape[0], page_scores.data_ptr(), max_pages,
            _p(status), _stream(q.device), kmeta=kmeta, page_scores=page_scores, status=status)
    return page_scores


def quest_select(q, kmeta, kv_indptr, kv_indices, token_budget: int, *, max_pages: int,
                 page_scores=None, cand_pages=None, cand_npages=None, status=None, counters=None
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Quest selector on stored page metadata (twilight/pyimpl/quest.py:17-122).

    Returns ``(cand_pages[B,H,max_k] int32 ascending, cand_npages[B,H] int32, page_scores)``.
    With ``counters`` (zeroed int32 ``[B*H_kv]``) scoring and selection run as one kernel."""
    q = _q3(q)
    b, hq, _ = q.shape
    n_total, hkv = kmeta.shape[0], kmeta.shape[1]
    max_k = max(1, token_budget // PAGE) + (1 if token_budget % PAGE else 0)
    max_k = min(max_k, max_pages)
    dev = q.device
    if page_scores is None:
        page_scores = torch.empty(b, hq, max_pages, dtype=torch.float32, device=dev)
    if cand_pages is None:
        cand_pages = torch.empty(b, hq, max_k, dtype=torch.int32, device=dev)
    if cand_npages is None:
        cand_npages = torch.empty(b, hq, dtype=torch.int32, device=dev)
    s = _stream(dev)
    if counters is not None:
        _launch("quest_select", q, q.data_ptr(), _dtype_code(q), kmeta.data_ptr(), kv_indptr.data_ptr(),
                kv_indices.data_ptr(), b, hq, hkv, n_total, token_budget, page_scores.data_ptr(), max_pages,
                cand_pages.data_ptr(), cand_npages.data_ptr(), cand_pages.shape[-1], counters.data_ptr(),
                _p(status), s, kmeta=kmeta, page_scores=page_scores, cand_pages=cand_pages, status=status)
        return cand_pages, cand_npages, page_scores
    _launch("quest_page_scores", q, q.data_ptr(), _dtype_code(q), kmeta.data_ptr(), kv_indptr.data_ptr(),
            kv_indices.data_ptr(), b, hq, hkv, n_total, page_scores.data_ptr(), max_pages, _p(status), s,
            kmeta=kmeta, page_scores=page_scores, status=status)
    _launch("quest_topk_pages", page_scores, page_scores.data_ptr(), max_pages, kv_indptr.data_ptr(), b, hq,
            token_budget, cand_pages.data_ptr(), cand_npages.data_ptr(), cand_pages.shape[-1], s,
            cand_pages=cand_pages, cand_npages=cand_npages)
    return cand_pages, cand_npages, page_scores


def quest_topk(page_scores, kv_indptr, token_budget: int, *, max_pages: int, cand_pages=None,
               cand_npages=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The selection half of :func:`quest_select` on given fp32 scores ``[B,H,max_pages]``:
    ascending positions of the ``max(1, budget//16) + (budget%16 != 0)`` best entries of each row
    (twilight/pyimpl/quest.py:93-99), ties to the lower position."""
    _cuda_contig(page_scores, "page_scores")
    b, hq, stride = page_scores.shape
    assert stride == max_pages and page_scores.dtype == torch.float32
    max_k = min(max(1, token_budget // PAGE) + (1 if token_budget % PAGE else 0), max_pages)
    dev = page_scores.device
    if cand_pages is None:
        cand_pages = torch.empty(b, hq, max_k, dtype=torch.int32, device=dev)
    if cand_npages is None:
        cand_npages = torch.empty(b, hq, dtype=torch.int32, device=dev)
    _launch("quest_topk_pages", page_scores, page_scores.data_ptr(), max_pages, kv_indptr.data_ptr(), b, hq,
            token_budget, cand_pages.data_ptr(), cand_npages.data_ptr(), cand_pages.shape[-1], _stream(dev),
            cand_pages=cand_pages, cand_npages=cand_npages)
    return cand_pages, cand_npages, page_scores


def estimate_int4(q, k4_pages, kv_indptr, kv_indices, kv_last_page_len, *, max_pages: int,
                  cand_pages=None, cand_npages=None, sm_scale: Optional[float] = None,
                  scores=None, variant: int = 0, status=None) -> torch.Tensor:
    """INT4 K-cache estimator (twilight/pyimpl/attention.py:247-255): fp32 scores
    ``[B,H,stride]``; slot s of a row is token ``cand_pages[s//16]*16+s%16`` (or token s when
    no candidate list is given)."""
    q = _q3(q)
    b, hq, _ = q.shape
    n_total, hkv = k4_pages.shape[0], k4_pages.shape[1]
    max_k = 0 if cand_pages is None else cand_pages.shape[-1]
    stride = (max_k if cand_pages is not None else max_pages) * PAGE
    if scores is None:
        scores = torch.empty(b, hq, stride, dtype=torch.float32, device=q.device)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    _launch("estimate_int4", q, q.data_ptr(), _dtype_code(q), k4_pages.data_ptr(), kv_indptr.data_ptr(),
            kv_indices.data_ptr(), kv_last_page_len.data_ptr(), _p(cand_pages), _p(cand_npages), max_k, b,
            hq, hkv, n_total, sm_scale, scores.data_ptr(), scores.shape[-1], variant, _p(status),
            _stream(q.device), k4_pages=k4_pages, scores=scores, cand_pages=cand_pages, status=status)
    return scores


def topp_prune(scores, kv_indptr, kv_last_page_len, top_p: Union[torch.Tensor, float], *,
               cand_pages=None, cand_npages=None, indices=None, budget=None, threshold=None,
               status=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 softmax + top-p search + compaction (twilight/pyimpl/top_p.py:10-15 and
    attention.py:280-285).  Returns ``(indices[B,H,stride] int32, budget[B,H] int32)``; the first
    ``budget`` entries of a row are the kept token positions in ascending order."""
    _cuda_contig(scores, "scores")
    b, hq, stride = scores.shape
    dev = scores.device
    if indices is None:
        indices = torch.empty(b, hq, stride, dtype=torch.int32, device=dev)
    if budget is None:
        budget = torch.empty(b, hq, dtype=torch.int32, device=dev)
    arr, val = (top_p, 0.0) if isinstance(top_p, torch.Tensor) else (None, float(top_p))
    if arr is not None:
        arr = arr.to(device=dev, dtype=torch.float32).contiguous()
    max_k = 0 if cand_pages is None else cand_pages.shape[-1]
    _launch("topp_prune", scores, scores.data_ptr(), stride, kv_indptr.data_ptr(),
            kv_last_page_len.data_ptr(), _p(cand_pages), _p(cand_npages), max_k, b, hq, _p(arr), val,
            indices.data_ptr(), indices.shape[-1], budget.data_ptr(), _p(threshold), _p(status),
            _stream(dev), indices=indices, budget=budget, cand_pages=cand_pages, status=status)
    return indices, budget


def threshold_prune(scores, kv_indptr, kv_last_page_len, threshold: float, *, cand_pages=None,
                    cand_npages=None, indices=None, budget=None, cut=None, status=None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Element-wise threshold pruner (twilight/pyimpl/elementwise_threshold.py:9-18) in index-list
    form: keeps candidates whose score exceeds ``score(token 0) - threshold``."""
    _cuda_contig(scores, "scores")
    b, hq, stride = scores.shape
    dev = scores.device
    if indices is None:
        indices = torch.empty(b, hq, stride, dtype=torch.int32, device=dev)
    if budget is None:
        budget = torch.empty(b, hq, dtype=torch.int32, device=dev)
    max_k = 0 if cand_pages is None else cand_pages.shape[-1]
    _launch("threshold_prune", scores, scores.data_ptr(), stride, kv_indptr.data_ptr(),
            kv_last_page_len.data_ptr(), _p(cand_pages), _p(cand_npages), max_k, b, hq, float(threshold),
            indices.data_ptr(), indices.shape[-1], budget.data_ptr(), _p(cut), _p(status), _stream(dev),
            indices=indices, budget=budget, cand_pages=cand_pages, status=status)
    return indices, budget


def prune_with_weights(scores, kv_indptr, kv_last_page_len, value, *, mode: str = "top_p",
                       cand_pages=None, cand_npages=None, indices=None, budget=None, weights=None,
                       threshold=None, status=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Top-p (``mode="top_p"``) or element-wise threshold (``mode="threshold"``) pruner that also
    returns, for every kept token, its un-normalised softmax weight over the estimated logits
    (for attention with ``use_estimated_weights_in_attn``, twilight/pyimpl/attention.py:295-296).
    Returns ``(indices, budget, weights[B,H,stride] fp32)``."""
    _cuda_contig(scores, "scores")
    b, hq, stride = scores.shape
    dev = scores.device
    if indices is None:
        indices = torch.empty(b, hq, stride, dtype=torch.int32, device=dev)
    if budget is None:
        budget = torch.empty(b, hq, dtype=torch.int32, device=dev)
    if weights is None:
        weights = torch.empty(b, hq, indices.shape[-1], dtype=torch.float32, device=dev)
    arr, val = (value, 0.0) if isinstance(value, torch.Tensor) else (None, float(value))
    if arr is not None:
        arr = arr.to(device=dev, dtype=torch.float32).contiguous()
    max_k = 0 if cand_pages is None else cand_pages.shape[-1]
    _launch("prune_with_weights", scores, {"top_p": 0, "threshold": 1}[mode], scores.data_ptr(), stride,
            kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), _p(cand_pages), _p(cand_npages), max_k, b,
            hq, _p(arr), val, indices.data_ptr(), indices.shape[-1], budget.data_ptr(), _p(threshold),
            weights.data_ptr(), _p(status), _stream(dev), indices=indices, budget=budget, weights=weights,
            status=status)
    return indices, budget, weights


def sparse_attn_workspace_bytes(batch: int, num_q_heads: int, index_stride: int, chunk: int = 256
                                ) -> int:
    return int(_lib.load().twl_sparse_attn_workspace_bytes(batch, num_q_heads, index_stride, chunk))


def sparse_decode_attn(q, k_pages, v_pages, kv_indptr, kv_indices, indices, budget, *,
                       sm_scale: Optional[float] = None, out=None, workspace=None,
                       chunk: int = 256, status=None, weights=None) -> torch.Tensor:
    """Attention of each (batch, query head) over its kept tokens
    (twilight/pyimpl/attention.py:188-190, :298-306).  Returns ``[B,H,D]`` in q's dtype.
    ``workspace``: zero-initialised uint8 tensor of ``sparse_attn_workspace_bytes`` bytes.
    ``weights`` (from :func:`prune_with_weights`): attend with these weights instead of exact
    q.k logits (attention.py:295-296); K is then not read."""
    q = _q3(q)
    b, hq, _ = q.shape
    n_total, hkv = k_pages.shape[0], k_pages.shape[1]
    stride = indices.shape[-1]
    if out is None:
        out = torch.empty(b, hq, HEAD_DIM, dtype=q.dtype, device=q.device)
    if workspace is None:
        workspace = torch.zeros(sparse_attn_workspace_bytes(b, hq, stride, chunk), dtype=torch.uint8,
                                device=q.device)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    if weights is not None:
        _launch("sparse_decode_attn_weighted", q, q.data_ptr(), _dtype_code(q), k_pages.data_ptr(),
                v_pages.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(), indices.data_ptr(), stride,
                budget.data_ptr(), weights.data_ptr(), b, hq, hkv, n_total, sm_scale, out.data_ptr(),
                workspace.data_ptr(), workspace.numel(), chunk, _p(status), _stream(q.device),
                k_pages=k_pages, v_pages=v_pages, out=out, workspace=workspace, indices=indices,
                status=status)
        return out
    _launch("sparse_decode_attn", q, q.data_ptr(), _dtype_code(q), k_pages.data_ptr(), v_pages.data_ptr(),
            kv_indptr.data_ptr(), kv_indices.data_ptr(), indices.data_ptr(), stride, budget.data_ptr(), b,
            hq, hkv, n_total, sm_scale, out.data_ptr(), workspace.data_ptr(), workspace.numel(), chunk,
            _p(status), _stream(q.device), k_pages=k_pages, v_pages=v_pages, out=out, workspace=workspace,
            indices=indices, status=status)
    return out


STATIC_ATTN_MAX_ROWS = 512


def sparse_decode_attn_static(q, k_pages, v_pages, kv_indptr, kv_indices, indices, budget, *,
                              out: torch.Tensor, sm_scale: Optional[float] = None, chunk: int = 256,
                              status=None) -> torch.Tensor:
    """:func:`sparse_decode_attn` on scratch memory that is part of the library itself, for
    callers that cannot allocate device memory after start-up (a process whose own pool holds all
    of it, a plugin called where allocation is forbidden).  ``out`` must be supplied; nothing is
    allocated here or in the library.  At most ``STATIC_ATTN_MAX_ROWS`` (batch x query heads) rows.
    All calls on a device share one scratch array, so calls that could overlap on the GPU must
    not be issued; make the first call on a device outside any stream capture."""
    q = _q3(q)
    b, hq, _ = q.shape
    n_total, hkv = k_pages.shape[0], k_pages.shape[1]
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    _launch("sparse_decode_attn_static", q, q.data_ptr(), _dtype_code(q), k_pages.data_ptr(),
            v_pages.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(), indices.data_ptr(),
            indices.shape[-1], budget.data_ptr(), b, hq, hkv, n_total, sm_scale, out.data_ptr(), chunk,
            _p(status), _stream(q.device), k_pages=k_pages, v_pages=v_pages, out=out, indices=indices,
            status=status)
    return out


def round_scores(scores: torch.Tensor, dtype: torch.dtype, post_scale: float = 1.0) -> torch.Tensor:
    """In place: ``scores <- round(round(scores) * post_scale)``, rounding to ``dtype`` (fp16/bf16), on
    an fp32 tensor.  Reproduces the model-dtype results of the reference's matmuls
    (twilight/pyimpl/quest.py:76-84, attention.py:252-254) on this library's fp32 scores."""
    _cuda_contig(scores, "scores")
    if scores.dtype != torch.float32:
        raise _lib.TwilightError("round_scores works on float32 scores")
    code = _dtype_code(torch.empty(0, dtype=dtype))
    _launch("round_scores", scores, scores.data_ptr(), scores.numel(), code, float(post_scale),
            _stream(scores.device))
    return scores


PRUNER_CODES = {"top_p": 0, "threshold": 1, "none": 2}
STEP_ESTIMATED_WEIGHTS, STEP_ROUND_TO_DTYPE = 1, 2


def step_workspace_layout(batch: int, num_q_heads: int, max_pages: int, token_budget: int,
                          attn_chunk: int = 256, flags: int = 0) -> "_lib.StepLayout":
    """Byte offsets of the parts of the one-buffer workspace of :func:`select_prune_attend_step`
    (``twl_step_workspace_layout``)."""
    lay = _lib.StepLayout()
    import ctypes
    _lib.check(_lib.load().twl_step_workspace_layout(batch, num_q_heads, max_pages, token_budget, attn_chunk,
                                                     flags, ctypes.addressof(lay)), "step_workspace_layout")
    return lay


def select_prune_attend_step(q, k_pages, v_pages, k4_pages, kmeta, kv_indptr, kv_indices, kv_last_page_len, *,
                             max_pages: int, token_budget: int, pruner: str, pruner_value: float,
                             out: torch.Tensor, workspace: torch.Tensor, top_p_arr=None,
                             sm_scale: Optional[float] = None, flags: int = 0, variant: int = 0,
                             attn_chunk: int = 256, status=None) -> torch.Tensor:
    """The decode step of one layer as ONE C-ABI call (``twl_select_prune_attend_step``): Quest
    selection when ``token_budget > 0``, INT4 estimate, pruner, sparse attention
    (twilight/pyimpl/attention.py:188-306).  ``workspace``: uint8 tensor of
    ``step_workspace_layout(...).total`` bytes, zeroed once after allocation."""
    q = _q3(q)
    b, hq, _ = q.shape
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(HEAD_DIM)
    arr = None
    if top_p_arr is not None:
        arr = top_p_arr.to(device=q.device, dtype=torch.float32).contiguous()
    _launch("select_prune_attend_step", q, q.data_ptr(), _dtype_code(q), k_pages.data_ptr(), v_pages.data_ptr(),
            k4_pages.data_ptr(), _p(kmeta), kv_indptr.data_ptr(), kv_indices.data_ptr(),
            kv_last_page_len.data_ptr(), b, hq, k_pages.shape[1], k_pages.shape[0], max_pages, token_budget,
            PRUNER_CODES[pruner], float(pruner_value), _p(arr), sm_scale, flags, variant, attn_chunk,
            out.data_ptr(), workspace.data_ptr(), workspace.numel(), _p(status), _stream(q.device),
            k_pages=k_pages, v_pages=v_pages, k4_pages=k4_pages, kmeta=kmeta, out=out, workspace=workspace,
            status=status, kv_indptr=kv_indptr, kv_indices=kv_indices)
    return out


# ---------------------------------------------------------------------------------------------
# cache-append side
# ---------------------------------------------------------------------------------------------
def quantize_k_pages(k_pages: torch.Tensor, k4_pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """K pages ``[P,Hkv,16,128]`` -> INT4 slabs ``[P,Hkv,1280]`` uint8, group 32
    (twilight/pyimpl/quantize.py:4-13 per group, arithmetic in the cache dtype)."""
    _cuda_contig(k_pages, "k_pages")
    p, hkv = k_pages.shape[0], k_pages.shape[1]
    if k4_pages is None:
        k4_pages = torch.empty(p, hkv, K4_SLAB_BYTES, dtype=torch.uint8, device=k_pages.device)
    _launch("quantize_k_pages", k_pages, k_pages.data_ptr(), _dtype_code(k_pages), k4_pages.data_ptr(),
            p * hkv, _stream(k_pages.device), k4_pages=k4_pages)
    return k4_pages


def build_page_meta(k_pages, kv_indptr, kv_indices, kv_last_page_len, *, max_pages: int,
                    kmeta: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Channel-wise (min,max) of every page ``[P,Hkv,2,128]`` (stored form of the chunk maxima of
    twilight/pyimpl/quest.py:39-74)."""
    _cuda_contig(k_pages, "k_pages")
    p, hkv = k_pages.shape[0], k_pages.shape[1]
    b = kv_indptr.numel() - 1
    if kmeta is None:
        kmeta = torch.zeros(p, hkv, 2, HEAD_DIM, dtype=k_pages.dtype, device=k_pages.device)
    _launch("build_page_meta", k_pages, k_pages.data_ptr(), _dtype_code(k_pages), kmeta.data_ptr(),
            kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr(), b, hkv, p, max_pages,
            _stream(k_pages.device), kmeta=kmeta)
    return kmeta


def append_kv(new_k, new_v, k_pages, v_pages, k4_pages, kmeta, kv_indptr, kv_indices,
              kv_last_page_len, status=None) -> None:
    """Writes one token per sequence (``new_k/new_v [B,Hkv,128]``) at the last position the page
    table describes, with its INT4 codes and the page metadata update."""
    _cuda_contig(new_k, "new_k")
    _cuda_contig(new_v, "new_v")
    b, hkv, _ = new_k.shape
    _launch("append_kv", new_k, new_k.data_ptr(), new_v.data_ptr(), _dtype_code(new_k), k_pages.data_ptr(),
            v_pages.data_ptr(), _p(k4_pages), _p(kmeta), kv_indptr.data_ptr(), kv_indices.data_ptr(),
            kv_last_page_len.data_ptr(), b, hkv, k_pages.shape[0], _p(status), _stream(new_k.device),
            k_pages=k_pages, v_pages=v_pages, k4_pages=k4_pages, kmeta=kmeta, status=status)


# ---------------------------------------------------------------------------------------------
# a prompt's way into the cache
# ---------------------------------------------------------------------------------------------
# rope_type: what its dictionary must hold, and what it may (those without an effect on the angles among them)
_LIMIT = "original_max_position_embeddings"
_ROPE_ENTRIES = {
    "default": ((), (_LIMIT,)),
    "linear": (("factor",), (_LIMIT,)),
    "dynamic": (("factor", _LIMIT), ()),
    "llama3": (("factor", _LIMIT, "low_freq_factor", "high_freq_factor"), ()),
    "yarn": (("factor", _LIMIT), ("attention_factor", "beta_fast", "beta_slow", "truncate")),
}


def rope_frequencies(rotary_dim: int = HEAD_DIM, base: float = 10000.0, *, scaling: Optional[dict] = None,
                     seq_len: Optional[int] = None, device="cuda") -> Tuple[torch.Tensor, float]:
    """Angles per position of the ``rotary_dim/2`` rotary pairs (float64, for :func:`rope_append_kv`) and the
    factor on cos and sin.  ``scaling`` takes the dictionaries that model configurations state
    (``rope_scaling``), by ``rope_type``: ``"default"``; ``"linear"`` (positions divided by ``factor``);
    ``"dynamic"`` (the base grows with ``seq_len`` beyond ``original_max_position_embeddings``); ``"llama3"``
    (long wavelengths divided by ``factor``, short ones kept, a ramp between) and ``"yarn"`` (the same in terms
    of the pair's index, with an attention factor; ``truncate: False`` keeps the ends of its ramp fractional).
    Entries that would change the angles and are not known here are refused."""
    if rotary_dim % 8 or not 8 <= rotary_dim <= HEAD_DIM:
        raise _lib.TwilightError(f"rotary_dim must be a multiple of 8 from 8 to {HEAD_DIM}")
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _ROPE_ENTRIES:
        raise _lib.TwilightError(f"unknown rope_type {kind!r}")
    if scaling is not None:
        needs, takes = _ROPE_ENTRIES[kind]
        missing = [n for n in needs if scaling.get(n) is None]
        if missing:
            raise _lib.TwilightError(f"scaling of rope_type {kind!r} lacks {', '.join(missing)}")
        known = {"rope_type", "type", "factor", "rope_theta", "partial_rotary_factor", *needs, *takes}
        other = [n for n, x in scaling.items() if n not in known and x is not None]
        # (a factor that states the whole attention scale makes the two that it is made of superfluous)
        if kind == "yarn" and scaling.get("attention_factor") is not None:
            other = [n for n in other if n not in ("mscale", "mscale_all_dim")]
        if other:
            raise _lib.TwilightError(f"scaling of rope_type {kind!r} has entries that are not supported: {', '.join(other)}")
        if scaling.get("rope_theta") is not None and float(scaling["rope_theta"]) != float(base):
            raise _lib.TwilightError(f"scaling states rope_theta {scaling['rope_theta']}, base is {base}")
        part = scaling.get("partial_rotary_factor")
        if part is not None and int(HEAD_DIM * part) != rotary_dim:
            raise _lib.TwilightError(f"scaling states partial_rotary_factor {part}, rotary_dim is {rotary_dim}")
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    factor = 1.0 if scaling is None or kind == "default" else float(scaling["factor"])
    attention_scale = 1.0
    if kind == "dynamic":
        limit = scaling[_LIMIT]
        n = max(limit, seq_len or limit)
        base = base * (factor * n / limit - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
    freqs = base ** (-pair / rotary_dim)
    if kind == "linear":
        freqs = freqs / factor
    elif kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = scaling[_LIMIT] * freqs / (2 * math.pi)  # within the original context
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freqs = freqs * (keep + (1 - keep) / factor)
    elif kind == "yarn":
        limit = scaling[_LIMIT]

        def index_of(turns):  # of the pair that makes this many turns within the original context
            return rotary_dim * math.log(limit / (turns * 2 * math.pi)) / (2 * math.log(base))
        first, last = index_of(float(scaling.get("beta_fast") or 32)), index_of(float(scaling.get("beta_slow") or 1))
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        ramp = ((pair / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
        freqs = freqs * (1 - ramp + ramp / factor)
        attention_scale = scaling.get("attention_factor")
        if attention_scale is None:
            attention_scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freqs.to(device), float(attention_scale)


def _cuda(t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise _lib.TwilightError("the operators take CUDA tensors only (there is no CPU path)")


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 3 or t.shape[2] != HEAD_DIM or t.stride(2) != 1:
        raise _lib.TwilightError(f"{name} must be [tokens, heads, {HEAD_DIM}] with contiguous heads")
    return t


# (These run on every call of operators that can take less than ten microseconds on the GPU: plain comparisons,
# messages only where one fails.)
def _pool(t: torch.Tensor, name: str, dtype: torch.dtype, shape) -> None:
    """A K/V pool (or its metadata): contiguous, of the queries' type and of the given shape."""
    if t.dtype != dtype:
        raise _lib.TwilightError(f"{name} is {t.dtype}, q is {dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise _lib.TwilightError(f"{name} must be contiguous {list(shape)} (pages and heads of k_pages)")


def _i32(t: torch.Tensor, name: str, entries: int = -1) -> int:
    """Checks a contiguous int32 tensor (of so many entries); its address."""
    if t.dtype != _INT32 or not t.is_contiguous():
        raise _lib.TwilightError(f"{name} must be contiguous int32")
    if entries >= 0 and t.numel() != entries:
        raise _lib.TwilightError(f"{name} must have {entries} entries")
    return t.data_ptr()


def _kv_pools(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor) -> Tuple[int, int]:
    """Checks the K and V pools against the queries; ``(pages, KV heads)``."""
    if k_pages.dim() != 4:
        raise _lib.TwilightError(f"k_pages must be [pages, kv heads, {PAGE}, {HEAD_DIM}]")
    pages, hkv, page, dim = k_pages.shape
    dtype = q.dtype
    if (page != PAGE or dim != HEAD_DIM or k_pages.dtype != dtype or not k_pages.is_contiguous() or v_pages.dtype != dtype
            or v_pages.shape != k_pages.shape or not v_pages.is_contiguous()):
        _pool(k_pages, "k_pages", dtype, (pages, hkv, PAGE, HEAD_DIM))  # (says which)
        _pool(v_pages, "v_pages", dtype, (pages, hkv, PAGE, HEAD_DIM))
    if hkv == 0 or q.shape[1] % hkv:
        raise _lib.TwilightError("query heads must be a multiple of KV heads")
    return pages, hkv


def rope_append_kv(q, k, v, freqs, k_pages, v_pages, k4_pages, kmeta, qo_indptr, kv_indptr, kv_indices,
                   kv_last_page_len, *, positions=None, interleaved: bool = False, attention_scale: float = 1.0,
                   out=None, status=None) -> torch.Tensor:
    """Rotary positions and the cache append of a ragged batch's new tokens in one pass; returns the rotated q.

    ``q [T,Hq,128]``, ``k, v [T,Hkv,128]`` (views of one fused projection will do): sequence b's new tokens are
    rows ``qo_indptr[b]:qo_indptr[b+1]`` and the last tokens of the sequence that the page table describes.
    ``freqs`` (from :func:`rope_frequencies`) rotates the first ``2*len(freqs)`` channels, as halves or
    ``interleaved`` pairs; None rotates nothing.  ``positions`` (int32 or int64 ``[T]``) replaces the cache
    positions.  K and V rows, INT4 slabs (``k4_pages``) and page metadata (``kmeta``) are written in place; the
    last two may be None.  ``out`` may be q itself."""
    _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    t, hq = q.shape[0], q.shape[1]
    batch = qo_indptr.numel() - 1
    pages, hkv = _kv_pools(q, k_pages, v_pages)
    if k.shape != (t, hkv, HEAD_DIM) or v.shape != (t, hkv, HEAD_DIM) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise _lib.TwilightError(f"k and v must have q's tokens and type and the cache's {hkv} heads")
    if kmeta is not None:
        _pool(kmeta, "kmeta", q.dtype, (pages, hkv, 2, HEAD_DIM))
    if k4_pages is not None:
        _pool(k4_pages, "k4_pages", torch.uint8, (pages, hkv, K4_SLAB_BYTES))
    qo_p, ptr_p = _i32(qo_indptr, "qo_indptr"), _i32(kv_indptr, "kv_indptr", batch + 1)
    idx_p, last_p = _i32(kv_indices, "kv_indices"), _i32(kv_last_page_len, "kv_last_page_len", batch)
    if freqs is not None and (freqs.dtype != torch.float64 or not freqs.is_contiguous()):
        raise _lib.TwilightError("freqs must be contiguous float64 (see rope_frequencies)")
    if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or positions.shape != (t,)
                                  or not positions.is_contiguous()):
        raise _lib.TwilightError("positions must be contiguous int32 or int64, one for each token")
    if out is None:
        out = torch.empty(t, hq, HEAD_DIM, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise _lib.TwilightError("out must have q's shape and type, and contiguous heads")
    _cuda(q)
    if t == 0:
        return out
    index = q.get_device()
    (q_ts, q_hs, _), (k_ts, k_hs, _), (v_ts, v_hs, _), (o_ts, o_hs, _) = q.stride(), k.stride(), v.stride(), out.stride()
    _launch_small("rope_append_kv", index,
                  ("k", k, "v", v, "out", out, "positions", positions, "freqs", freqs, "k_pages", k_pages, "v_pages", v_pages,
                   "k4_pages", k4_pages, "kmeta", kmeta, "qo_indptr", qo_indptr, "kv_indptr", kv_indptr,
                   "kv_indices", kv_indices, "kv_last_page_len", kv_last_page_len, "status", status),
                  (q.data_ptr(), k.data_ptr(), v.data_ptr(), _dtype_code(q), q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, out.data_ptr(),
                   o_ts, o_hs, _p(positions), 0 if positions is None else positions.dtype == torch.int64, _p(freqs),
                   0 if freqs is None else 2 * freqs.numel(), interleaved, attention_scale, k_pages.data_ptr(),
                   v_pages.data_ptr(), _p(k4_pages), _p(kmeta), qo_p, ptr_p, idx_p, last_p, t, batch, hq, hkv, pages,
                   _p(status), torch._C._cuda_getCurrentRawStream(index)))
    return out


def dequantize_k_pages(k4_pages, page_ids=None, *, dtype: torch.dtype, out=None, status=None) -> torch.Tensor:
    """Values of INT4 slabs, ``code*scale + minimum`` rounded to ``dtype``: ``[n,Hkv,16,128]`` of the pages
    ``page_ids`` (int32 ``[n]``), or of every page."""
    _cuda_contig(k4_pages, "k4_pages")
    if k4_pages.dtype != torch.uint8 or k4_pages.dim() != 3 or k4_pages.shape[2] != K4_SLAB_BYTES:
        raise _lib.TwilightError(f"k4_pages must be uint8 [pages, kv heads, {K4_SLAB_BYTES}]")
    pages, hkv = k4_pages.shape[0], k4_pages.shape[1]
    if page_ids is not None and (page_ids.dtype != torch.int32 or page_ids.dim() != 1 or not page_ids.is_contiguous()):
        raise _lib.TwilightError("page_ids must be contiguous int32 [n]")
    n = pages if page_ids is None else page_ids.numel()
    if out is None:
        out = torch.empty(n, hkv, PAGE, HEAD_DIM, dtype=dtype, device=k4_pages.device)
    elif out.shape != (n, hkv, PAGE, HEAD_DIM) or out.dtype != dtype or not out.is_contiguous():
        raise _lib.TwilightError(f"out must be contiguous {dtype} [{n}, {hkv}, {PAGE}, {HEAD_DIM}]")
    if out.numel() == 0:
        return out
    index = k4_pages.get_device()
    _launch_small("dequantize_k_pages", index, ("page_ids", page_ids, "out", out, "status", status),
                  (k4_pages.data_ptr(), _p(page_ids), n, out.data_ptr(), _dtype_code(out), hkv, pages, _p(status),
                   torch._C._cuda_getCurrentRawStream(index)))
    return out


# ---------------------------------------------------------------------------------------------
# attention of more than one token at a time
# ---------------------------------------------------------------------------------------------
def _queries(q: torch.Tensor) -> None:
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.stride(2) != 1 or (q.stride(1) != HEAD_DIM and q.shape[1] > 1):
        raise _lib.TwilightError(f"q must be [tokens, heads, {HEAD_DIM}], the heads of a token contiguous")


def _result(q: torch.Tensor, out, lse) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Checked or fresh output, and the log-sum-exp buffer where one is wanted (``lse``: True or a tensor)."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise _lib.TwilightError("out must be contiguous, of q's shape and type")
    if lse is None or lse is False:
        return out, None
    if lse is True:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    elif lse.shape != q.shape[:2] or lse.dtype != torch.float32 or not lse.is_contiguous():
        raise _lib.TwilightError("lse must be contiguous float32 [tokens, query heads]")
    return out, lse


def _workspace(t: Optional[torch.Tensor], nbytes: int, device) -> torch.Tensor:
    if t is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if t.dtype != torch.uint8 or not t.is_contiguous():
        raise _lib.TwilightError("workspace must be contiguous uint8")
    return t


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name: str, index: int, *sizes: int) -> int:
    """(The sizes follow the GPU's SM count: asked with the device current that the call runs on.)"""
    fn = getattr(_lib.load(), f"twl_{name}_workspace_bytes")
    if index < 0:
        return int(fn(*sizes))
    with torch.cuda.device(index):
        return int(fn(*sizes))


def _device_index(device) -> int:
    """The device's index, the current one's for None; -1 where there is none."""
    index = None if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device() if torch.cuda.is_available() else -1
    return index


def prompt_attn_workspace_bytes(num_tokens: int, batch: int, num_q_heads: int, num_kv_heads: int, max_pages: int,
                                query_block: int = 0, *, device=None) -> int:
    """Bytes of :func:`prompt_attn`'s workspace on ``device`` (None: the current one); ``query_block`` is 0 without block
    lists."""
    return _workspace_bytes("prompt_attn", _device_index(device), num_tokens, batch, num_q_heads, num_kv_heads, max_pages,
                            query_block)


def prompt_attn(q, k_pages, v_pages, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, *, max_pages: int,
                causal: bool = True, block_pages=None, block_npages=None, query_block: int = 64,
                sm_scale: Optional[float] = None, out=None, lse=None, workspace=None, status=None):
    """Attention of a ragged batch's new tokens over the paged cache: whole prompts, chunks of them, or a few tokens
    to verify (the dense prefill of twilight/pyimpl/attention.py:157-182, on pages).

    ``q [T,Hq,128]``: sequence b's queries are rows ``qo_indptr[b]:qo_indptr[b+1]`` and the last tokens that its page
    table describes (append them first, :func:`rope_append_kv`).  ``block_pages``/``block_npages`` from
    :func:`quest_select_blocks` restrict every block of ``query_block`` queries to its pages.  ``max_pages``: the
    largest page count of a sequence.  Returns ``out [T,Hq,128]``, and with ``lse`` (True or a tensor) also the fp32
    ``[T,Hq]`` logarithms of the sums of exponentials.  ``workspace``: ``prompt_attn_workspace_bytes`` bytes, one for
    each call that may overlap with another.  V must be finite also where a query does not see its token (its weight is
    zero there); rows behind a sequence's end may hold anything."""
    _queries(q)
    t, hq = q.shape[0], q.shape[1]
    pages, hkv = _kv_pools(q, k_pages, v_pages)
    batch = qo_indptr.numel() - 1
    qo_p, ptr_p = _i32(qo_indptr, "qo_indptr"), _i32(kv_indptr, "kv_indptr", batch + 1)
    idx_p, last_p = _i32(kv_indices, "kv_indices"), _i32(kv_last_page_len, "kv_last_page_len", batch)
    out, lse = _result(q, out, lse)
    if (block_pages is None) != (block_npages is None):
        raise _lib.TwilightError("block_pages and block_npages go together")
    max_k = 0
    if block_pages is not None:
        _i32(block_pages, "block_pages")
        _i32(block_npages, "block_npages")
        slots, max_k = t // query_block + batch, block_pages.shape[-1]
        if block_pages.shape != (slots, hkv, max_k) or block_npages.shape != (slots, hkv):
            raise _lib.TwilightError(f"block_pages must be [{slots}, {hkv}, max_k], block_npages [{slots}, {hkv}]")
    else:
        query_block = 0
    _cuda(q)
    if t > 0:
        index = q.get_device()
        workspace = _workspace(workspace, _workspace_bytes("prompt_attn", index, t, batch, hq, hkv, max_pages, query_block),
                               q.device)
        _launch_small("prompt_attn", index,
                      ("k_pages", k_pages, "v_pages", v_pages, "qo_indptr", qo_indptr, "kv_indptr", kv_indptr,
                       "kv_indices", kv_indices, "kv_last_page_len", kv_last_page_len, "block_pages", block_pages,
                       "block_npages", block_npages, "out", out, "lse", lse, "workspace", workspace, "status", status),
                      (q.data_ptr(), _dtype_code(q), q.stride(0), k_pages.data_ptr(), v_pages.data_ptr(), qo_p, ptr_p, idx_p,
                       last_p, t, batch, hq, hkv, pages, max_pages, causal, _p(block_pages), _p(block_npages), max_k,
                       query_block, _SM_SCALE if sm_scale is None else sm_scale, out.data_ptr(), _p(lse),
                       workspace.data_ptr(), workspace.numel(), _p(status), torch._C._cuda_getCurrentRawStream(index)))
    return out if lse is None else (out, lse)


def quest_select_blocks(q, kmeta, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, token_budget: int, *,
                        max_pages: int, query_block: int = 64, block_pages=None, block_npages=None, pooled=None,
                        page_scores=None, status=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Pages that every block of ``query_block`` queries (a multiple of 16) of a prompt attends to, for
    :func:`prompt_attn`: all from the page of its first position on, and of those before it the token budget's best
    by the sum of Quest's bounds over the block's rows (twilight/pyimpl/quest.py:37-99 applied to a block), as 64-bit
    sums would choose them, ties to the lower page.

    Returns ``(block_pages [slots,Hkv,max_k] int32 ascending, block_npages [slots,Hkv] int32)`` with
    ``slots = T//query_block + batch``; block j of sequence b is row ``qo_indptr[b]//query_block + b + j``, rows without a
    block have a count of 0.  ``max_pages``: the largest page count of a sequence (pages behind it are left out, and
    flagged in ``status``, as sequences are whose entries make no sense)."""
    _queries(q)
    t, hq = q.shape[0], q.shape[1]
    batch = qo_indptr.numel() - 1
    if kmeta.dim() != 4:
        raise _lib.TwilightError(f"kmeta must be [pages, kv heads, 2, {HEAD_DIM}]")
    hkv = kmeta.shape[1]
    _pool(kmeta, "kmeta", q.dtype, (kmeta.shape[0], hkv, 2, HEAD_DIM))
    if hkv == 0 or hq % hkv:
        raise _lib.TwilightError("query heads must be a multiple of KV heads")
    _i32(qo_indptr, "qo_indptr")
    _i32(kv_indptr, "kv_indptr", batch + 1)
    _i32(kv_indices, "kv_indices")
    _i32(kv_last_page_len, "kv_last_page_len", batch)
    if token_budget <= 0 or max_pages <= 0:
        raise _lib.TwilightError("token_budget and max_pages must be positive")
    if query_block < PAGE or query_block % PAGE:
        raise _lib.TwilightError(f"query_block must be a multiple of {PAGE}")
    _cuda(q)
    slots = t // query_block + batch
    # a block that starts inside a page lies in one page more than its tokens fill
    max_k = min(max(1, token_budget // PAGE) + (1 if token_budget % PAGE else 0) + query_block // PAGE + 1, max_pages)
    dev = q.device
    if block_pages is None:
        block_pages = torch.empty(slots, hkv, max_k, dtype=torch.int32, device=dev)
    if block_npages is None:
        block_npages = torch.empty(slots, hkv, dtype=torch.int32, device=dev)
    if pooled is None:
        pooled = torch.empty(slots, hkv, 2 * HEAD_DIM, dtype=torch.float32, device=dev)
    if page_scores is None:
        page_scores = torch.empty(slots, hkv, max_pages, dtype=torch.float32, device=dev)
    _i32(block_pages, "block_pages")
    _i32(block_npages, "block_npages")
    if block_pages.dim() != 3 or block_pages.shape[:2] != (slots, hkv) or block_pages.shape[2] < max_k \
            or block_npages.shape != (slots, hkv):
        raise _lib.TwilightError(f"block_pages must be [{slots}, {hkv}, at least {max_k}], block_npages [{slots}, {hkv}]")
    for name, x, width in (("pooled", pooled, 2 * HEAD_DIM), ("page_scores", page_scores, max_pages)):
        if x.shape != (slots, hkv, width) or x.dtype != torch.float32 or not x.is_contiguous():
            raise _lib.TwilightError(f"{name} must be contiguous float32 [{slots}, {hkv}, {width}]")
    if t > 0:
        _launch("quest_select_blocks", q, q.data_ptr(), _dtype_code(q), q.stride(0), kmeta.data_ptr(),
                qo_indptr.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_last_page_len.data_ptr(), t, batch,
                hq, hkv, kmeta.shape[0], token_budget, query_block, max_pages, pooled.data_ptr(), page_scores.data_ptr(),
                block_pages.data_ptr(), block_npages.data_ptr(), block_pages.shape[2], _p(status), _stream(dev),
                kmeta=kmeta, qo_indptr=qo_indptr, kv_indptr=kv_indptr, kv_indices=kv_indices,
                kv_last_page_len=kv_last_page_len, pooled=pooled, page_scores=page_scores, block_pages=block_pages,
                block_npages=block_npages, status=status)
    return block_pages, block_npages


def shared_prefix_workspace_bytes(batch: int, num_groups: int, num_q_heads: int, num_kv_heads: int, max_pages: int, *,
                                  device=None) -> int:
    """Bytes of :func:`shared_prefix_attn`'s workspace on ``device`` (None: the current one)."""
    return _workspace_bytes("shared_prefix", _device_index(device), batch, num_groups, num_q_heads, num_kv_heads, max_pages)


def shared_prefix_attn(q, k_pages, v_pages, group_indptr, prefix_indptr, prefix_indices, prefix_last_page_len, kv_indptr,
                       kv_indices, kv_last_page_len, *, max_pages: Optional[int] = None, sm_scale: Optional[float] = None,
                       out=None, lse=None, workspace=None, status=None):
    """Decode attention of groups of sequences over a prefix that a group shares (read once for the whole group) and
    each sequence's own pages behind it.

    ``q [B,Hq,128]`` (or ``[B,Hq,1,128]``), one token per sequence.  Group i is sequences
    ``group_indptr[i]:group_indptr[i+1]``; the three ``prefix_*`` tensors are its page table, the three ``kv_*``
    tensors that of the sequences' own parts (no pages: nothing of its own).  ``max_pages``: the largest page count of
    any of them; None takes the lengths of the index lists, which is an upper bound.  Returns ``out [B,Hq,128]``, and
    with ``lse`` also the fp32 ``[B,Hq]`` logarithms of the sums of exponentials."""
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise _lib.TwilightError("decode step only: q_len must be 1")
        q = q[:, :, 0, :]
    _queries(q)
    b, hq = q.shape[0], q.shape[1]
    pages, hkv = _kv_pools(q, k_pages, v_pages)
    groups = group_indptr.numel() - 1
    group_p, pptr_p = _i32(group_indptr, "group_indptr"), _i32(prefix_indptr, "prefix_indptr", groups + 1)
    pidx_p = _i32(prefix_indices, "prefix_indices")
    plast_p = _i32(prefix_last_page_len, "prefix_last_page_len", groups)
    ptr_p, idx_p = _i32(kv_indptr, "kv_indptr", b + 1), _i32(kv_indices, "kv_indices")
    last_p = _i32(kv_last_page_len, "kv_last_page_len", b)
    if groups < 1:
        raise _lib.TwilightError("group_indptr must have at least two entries")
    out, lse = _result(q, out, lse)
    _cuda(q)
    if b > 0:
        if max_pages is None:
            max_pages = max(prefix_indices.numel(), kv_indices.numel(), 1)
        index = q.get_device()
        workspace = _workspace(workspace, _workspace_bytes("shared_prefix", index, b, groups, hq, hkv, max_pages), q.device)
        _launch_small("shared_prefix_attn", index,
                      ("k_pages", k_pages, "v_pages", v_pages, "group_indptr", group_indptr, "prefix_indptr", prefix_indptr,
                       "prefix_indices", prefix_indices, "prefix_last_page_len", prefix_last_page_len, "kv_indptr", kv_indptr,
                       "kv_indices", kv_indices, "kv_last_page_len", kv_last_page_len, "out", out, "lse", lse,
                       "workspace", workspace, "status", status),
                      (q.data_ptr(), _dtype_code(q), q.stride(0), k_pages.data_ptr(), v_pages.data_ptr(), group_p, pptr_p,
                       pidx_p, plast_p, ptr_p, idx_p, last_p, b, groups, hq, hkv, pages, max_pages,
                       _SM_SCALE if sm_scale is None else sm_scale, out.data_ptr(), _p(lse), workspace.data_ptr(),
                       workspace.numel(), _p(status), torch._C._cuda_getCurrentRawStream(index)))
    return out if lse is None else (out, lse)


def indices_to_mask(indices, budget, seq_len: int) -> torch.Tensor:
    """Index lists -> the reference's mask layout ``bool[B,H,1,L]`` (attention.py:199-281)."""
    b, hq, stride = indices.shape
    mask = torch.zeros(b, hq, 1, seq_len, dtype=torch.bool, device=indices.device)
    _launch("indices_to_mask", indices, indices.data_ptr(), stride, budget.data_ptr(), b * hq,
            mask.data_ptr(), seq_len, _stream(indices.device), budget=budget, mask=mask)
    return mask


def batched_sparse_gemv_int4_k(q, o, k_cache_int4, quant_scales, quant_zeros, kv_page_indices,
                               kv_page_indptr, kv_last_page_len):
    """Same name and argument order as the absent ``ftka.cuda_ops.gemv`` op called at
    benchmark/efficiency/bench_gemv.py:445-454: raw ``q.k`` (no 1/sqrt(D)) of every token of
    every sequence written into ``o [B,H,L]``.  Differences, all forced by the group-32 cache:
    ``k_cache_int4`` is the slab tensor ``[P,Hkv,1280]`` that already carries scale and minimum,
    so ``quant_scales``/``quant_zeros`` must be ``None``; page size is 16; ``o`` is fp32 and its
    last dimension a multiple of 16."""
    if quant_scales is not None or quant_zeros is not None:
        raise _lib.TwilightError("scale/min live inside the INT4 slabs; pass None for both")
    if o.dtype != torch.float32 or o.shape[-1] % PAGE:
        raise _lib.TwilightError("o must be float32 with a last dimension that is a multiple of 16")
    estimate_int4(q, k_cache_int4, kv_page_indptr, kv_page_indices, kv_last_page_len,
                  max_pages=o.shape[-1] // PAGE, sm_scale=1.0, scores=o)
    return o
