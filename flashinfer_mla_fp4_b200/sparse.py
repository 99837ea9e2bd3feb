"""Sparse FP4 MLA decode: attention over the pages that a cheap score selects for each query.

A long request's decode step reads all of its cache for a few pages that matter.  Here every full page has a *summary*, its mean
key in 8 bits (576 codes and one FP32 scale, a 36th of a page of 64 tokens), a query scores the summaries, and attention runs over
the best pages alone.  The reference has no counterpart: it attends to whole requests.

* ``summarize_pages`` / ``summarize_new_pages``  summaries of pages by number, or of those that a step's new tokens have filled;
* ``select_pages``                               for each query position a block table of ``budget`` pages and the length to go with it;
* ``BatchMLASparseDecodeFP4Wrapper``             selection and attention as ``plan()/run()``;
* ``SparsePages``                                the choice of budget that ``FP4MLADecodeBackend(sparse=...)`` takes.

Summary.  With a page's n token scales s_t, latent values e_td and RoPE values r_td, S = max |s_t| and w_t = round(32767 s_t / S):
latent mean S / (32767 n) sum_t w_t e_td, RoPE mean 1/n sum_t r_td, scale = max |mean| / 127, code = round(mean / scale).  A page with a token
scale that is not finite or a NaN among its RoPE values has the scale NaN.

Selection.  Of a request with no more than ``budget`` pages all of them; else the first ``sink_pages``, the last ``local_pages`` (the page that
is not full among them) and the pages of the best score max_h <q_h, mean>, with the heads of the query as integers of their largest
binade's 1/64: NaN first, ties to the page nearer the start.  Dots are of integers, so the same pages come out on every GPU and run.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _cabi
from .api_log import api_logged
from .kvcache import HEAD_DIM_QK, ROW_BYTES
from .wrapper import BatchMLADecodeCuteDSLFP4Wrapper, validate_page_ids

PAGE_SIZES = (8, 16, 32, 64, 128)
_INT32 = 2**31 - 1  # counts are handed to the kernels in 32 bits
_native = _cabi.native


@dataclass(frozen=True)
class SparsePages:
    """How many pages a query attends to: ``budget_pages`` in all, the first ``sink_pages`` and the last ``local_pages`` always."""

    budget_pages: int
    sink_pages: int = 1
    local_pages: int = 2
    causal: bool = False

    def __post_init__(self) -> None:
        if self.budget_pages > _INT32:
            raise ValueError(f"budget_pages must be below 2^31, got {self.budget_pages}")
        if self.sink_pages < 0 or self.local_pages < 1 or self.sink_pages + self.local_pages > self.budget_pages:
            raise ValueError(f"sink_pages ({self.sink_pages}) must not be negative, local_pages ({self.local_pages}) at least 1, and their "
                             f"sum within budget_pages ({self.budget_pages})")


def check_tensor(name: str, t, dtype: torch.dtype, shape, device) -> None:
    """ValueError unless `t` is a contiguous tensor of that dtype and shape on that device (None in the shape: any extent)."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != len(shape) or not t.is_contiguous() or any(
            n is not None and t.shape[i] != n for i, n in enumerate(shape)):
        said = f"{t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple('*' if n is None else n for n in shape)}, got {said}")
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}, got {t.device}")


def check_tables(block_tables, seq_lens, device, batch: Optional[int] = None) -> None:
    if not isinstance(block_tables, torch.Tensor) or block_tables.dtype != torch.int32 or block_tables.dim() != 2 or (
            block_tables.shape[1] > 0 and block_tables.stride(1) != 1) or block_tables.stride(0) < 0:
        raise ValueError("block_tables must be an int32 [batch, max_pages] tensor with unit inner stride")
    if max(block_tables.shape) > _INT32:
        raise ValueError(f"block_tables must have fewer than 2^31 rows and pages a row, got {tuple(block_tables.shape)}")
    if not block_tables.is_cuda or block_tables.device != device:
        raise ValueError(f"block_tables must be a CUDA tensor on {device}, got {block_tables.device}")
    if batch is not None and block_tables.shape[0] != batch:
        raise ValueError("block_tables must have one row per request")
    check_tensor("seq_lens", seq_lens, torch.int32, (block_tables.shape[0],), device)


def check_cache(kv_cache, kv_cache_sf) -> Tuple[int, int]:
    """(pages, page size) of the two cache tensors; ValueError for what is not a cache."""
    if not isinstance(kv_cache, torch.Tensor) or kv_cache.dim() != 3 or kv_cache.shape[2] != ROW_BYTES or kv_cache.shape[1] not in PAGE_SIZES:
        raise ValueError(f"kv_cache must have shape [pages, page_size, {ROW_BYTES}] with a page_size of {PAGE_SIZES}")
    if not kv_cache.is_cuda:
        raise ValueError(f"kv_cache must be a CUDA tensor, got {kv_cache.device}")
    pages, page_size = kv_cache.shape[:2]
    check_tensor("kv_cache", kv_cache, torch.uint8, (None, None, ROW_BYTES), kv_cache.device)
    check_tensor("kv_cache_sf", kv_cache_sf, torch.float32, (pages, page_size, 1), kv_cache.device)
    return pages, page_size


def check_summary(summary, summary_sf, pages: Optional[int], device) -> int:
    check_tensor("summary", summary, torch.int8, (pages, HEAD_DIM_QK), device)
    check_tensor("summary_sf", summary_sf, torch.float32, (summary.shape[0],), device)
    return summary.shape[0]


@api_logged
def summarize_pages(kv_cache: torch.Tensor, kv_cache_sf: torch.Tensor, summary: torch.Tensor, summary_sf: torch.Tensor,
                    page_ids: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
    """Write the summaries of full pages: ``summary`` int8 [pages, 576] and ``summary_sf`` f32 [pages], at the numbers in ``page_ids``
    (int32, contiguous, on the device; those outside the pool are skipped, one that is named twice is written twice alike).

    All ``page_size`` rows of a page enter its summary, so call it for pages that are full.  ``status`` (int32 [8], zeroed) gets the error of a
    device-side wait that ran out.  Asynchronous on the current stream."""
    if _native.summarize(kv_cache, kv_cache_sf, summary, summary_sf, page_ids, None, None, 0, status):
        return  # the common form, checked and launched natively; otherwise nothing was done
    pages, page_size = check_cache(kv_cache, kv_cache_sf)
    dev = kv_cache.device
    check_summary(summary, summary_sf, pages, dev)
    check_tensor("page_ids", page_ids, torch.int32, (None,), dev)
    if status is not None:
        check_tensor("status", status, torch.int32, (8,), dev)
    if page_ids.numel() == 0:
        return
    with torch.cuda.device(dev):
        _cabi.check(_cabi.lib.mla_fp4_summarize_pages(kv_cache.data_ptr(), kv_cache_sf.data_ptr(), pages, page_size, page_ids.data_ptr(),
                                                      page_ids.numel(), summary.data_ptr(), summary_sf.data_ptr(),
                                                      None if status is None else status.data_ptr(), torch.cuda.current_stream(dev).cuda_stream))


@api_logged
def summarize_new_pages(kv_cache: torch.Tensor, kv_cache_sf: torch.Tensor, summary: torch.Tensor, summary_sf: torch.Tensor,
                        block_tables: torch.Tensor, seq_lens: torch.Tensor, new_tokens: int, status: Optional[torch.Tensor] = None) -> None:
    """Write the summaries of the pages that the newest ``new_tokens`` tokens of each request have filled.

    ``seq_lens`` (int32 [batch]) counts the new tokens, ``block_tables`` int32 [batch, max_pages].  What a step calls behind
    ``write_tokens``; a page that the step has not filled is left alone.  Asynchronous on the current stream."""
    if _native.summarize(kv_cache, kv_cache_sf, summary, summary_sf, None, block_tables, seq_lens, new_tokens, status):
        return
    pages, page_size = check_cache(kv_cache, kv_cache_sf)
    dev = kv_cache.device
    check_summary(summary, summary_sf, pages, dev)
    check_tables(block_tables, seq_lens, dev)
    if new_tokens < 0:
        raise ValueError(f"new_tokens must not be negative, got {new_tokens}")
    if status is not None:
        check_tensor("status", status, torch.int32, (8,), dev)
    batch, width = block_tables.shape
    if batch == 0 or width == 0 or new_tokens == 0:
        return
    with torch.cuda.device(dev):
        _cabi.check(_cabi.lib.mla_fp4_summarize_new_pages(
            kv_cache.data_ptr(), kv_cache_sf.data_ptr(), pages, page_size, block_tables.data_ptr(), block_tables.stride(0), width,
            seq_lens.data_ptr(), batch, min(int(new_tokens), _INT32), summary.data_ptr(), summary_sf.data_ptr(),
            None if status is None else status.data_ptr(), torch.cuda.current_stream(dev).cuda_stream))


@api_logged
def select_pages(q: torch.Tensor, summary: torch.Tensor, summary_sf: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                 page_size: int, budget_pages: int, *, sink_pages: int = 1, local_pages: int = 2, causal: bool = False,
                 selected: Optional[torch.Tensor] = None, selected_lens: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages that each query position attends to: ``(selected, selected_lens)``, int32 [batch * q_len, budget_pages] and
    [batch * q_len], a block table and lengths for a decode step of batch * q_len requests of one query position.

    ``q`` e4m3 [batch, q_len, H, 576] (strides that are multiples of 16, unit inner stride, H <= 128); ``seq_lens`` int32 [batch].  With ``causal``
    position i of q_len does not see the q_len - 1 - i newest tokens; without it every position sees all of them, as in
    ``BatchMLADecodeCuteDSLFP4Wrapper.run``.  Entries behind a row's last page are 0.  ``workspace`` (int8, ``4 * batch * q_len`` times
    max_pages rounded up to a multiple of four; 16-byte aligned; allocated when not given) holds the scores.  ``status`` (int32 [8], zeroed) gets the error of
    a device-side wait that ran out: the pages are then some of the request's, but not the best.  Asynchronous on the current stream, capturable."""
    done = _native.select(q, summary, summary_sf, block_tables, seq_lens, page_size, budget_pages, sink_pages, local_pages, causal,
                          selected, selected_lens, workspace, status)
    if done is not None:
        return done
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[-1] != HEAD_DIM_QK or q.dtype != torch.float8_e4m3fn:
        raise ValueError(f"q must be an E4M3 tensor [batch, q_len, num_heads, {HEAD_DIM_QK}]")
    if not q.is_cuda:
        raise ValueError(f"q must be a CUDA tensor, got {q.device}")
    if q.stride(-1) != 1:
        raise ValueError("q must have unit stride in its last dimension")
    dev = q.device
    batch, q_len, heads, _ = q.shape
    if page_size not in PAGE_SIZES:
        raise ValueError(f"Unsupported page_size={page_size}: must be one of {PAGE_SIZES}")
    if q_len < 1 or not 1 <= heads <= 128:
        raise ValueError(f"q must have at least one query position and 1 to 128 heads, got {tuple(q.shape)}")
    causal = bool(causal)
    SparsePages(budget_pages, sink_pages, local_pages)  # (its checks)
    pages = check_summary(summary, summary_sf, None, dev)
    check_tables(block_tables, seq_lens, dev, batch)
    rows, width = batch * q_len, block_tables.shape[1]
    if selected is None:
        selected = torch.empty(rows, budget_pages, dtype=torch.int32, device=dev)
    else:
        check_tensor("selected", selected, torch.int32, (rows, budget_pages), dev)
    if selected_lens is None:
        selected_lens = torch.empty(rows, dtype=torch.int32, device=dev)
    else:
        check_tensor("selected_lens", selected_lens, torch.int32, (rows,), dev)
    need = _cabi.select_workspace_bytes(batch, q_len, width) if width > budget_pages else 0
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.int8, device=dev)
    else:
        check_tensor("workspace", workspace, torch.int8, (None,), dev)
        if workspace.numel() < need:
            raise ValueError(f"workspace has {workspace.numel()} bytes, but {need} are required")
    if status is not None:
        check_tensor("status", status, torch.int32, (8,), dev)
    if rows == 0:
        return selected, selected_lens
    a = _cabi.SelectArgs()
    a.q = q.data_ptr()
    a.q_stride_batch, a.q_stride_qpos, a.q_stride_head = q.stride(0), q.stride(1), q.stride(2)
    a.summary, a.summary_sf, a.num_pages = summary.data_ptr(), summary_sf.data_ptr(), pages
    a.block_tables, a.block_table_stride, a.seq_lens = block_tables.data_ptr(), block_tables.stride(0), seq_lens.data_ptr()
    a.selected, a.selected_lens = selected.data_ptr(), selected_lens.data_ptr()
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    a.batch, a.q_len, a.num_heads, a.page_size, a.width = batch, q_len, heads, page_size, width
    a.budget, a.sink_pages, a.local_pages, a.causal = budget_pages, sink_pages, local_pages, int(causal)
    a.status = None if status is None else status.data_ptr()
    with torch.cuda.device(dev):
        a.stream = torch.cuda.current_stream(dev).cuda_stream
        _cabi.check(_cabi.lib.mla_fp4_select_pages(C.byref(a)))
    return selected, selected_lens


class BatchMLASparseDecodeFP4Wrapper:
    """Sparse counterpart of ``BatchMLADecodeCuteDSLFP4Wrapper``: ``plan()`` once, ``run()`` per step.

    The workspace buffer (int8, on the device, borrowed) holds the decode step's scratch (``planner.workspace_bytes``), then the selection's
    table, lengths and scores (``workspace_bytes``).  Steps on several streams, and graphs that replay at the same time, need a wrapper and a
    workspace each.
    """

    def __init__(self, workspace_buffer: torch.Tensor) -> None:
        self._dense = BatchMLADecodeCuteDSLFP4Wrapper(workspace_buffer)
        self._workspace_buffer = workspace_buffer
        self._device = workspace_buffer.device
        self._pages: Optional[SparsePages] = None

    @api_logged
    def plan(self, num_heads: int, page_size: int, budget_pages: int, sink_pages: int = 1, local_pages: int = 2, causal: bool = False,
             out_dtype: Optional[torch.dtype] = None, variant=None, enable_pdl: Optional[bool] = None, max_ctas: Optional[int] = None) -> None:
        """Validate and bind the configuration.  ``causal``: position i of q_len does not see the q_len - 1 - i newest tokens.  The other
        arguments are those of ``SparsePages`` and of the dense wrapper's ``plan``; ``max_ctas`` caps the attention's grid and with it the partials, not
        the selection's, which takes up to two CTAs an SM for the scores and one a query position after them."""
        pages = SparsePages(budget_pages, sink_pages, local_pages, bool(causal))
        self._dense.plan(num_heads=num_heads, page_size=page_size, out_dtype=out_dtype, variant=variant, enable_pdl=enable_pdl, max_ctas=max_ctas)
        self._pages, self._num_heads, self._page_size = pages, num_heads, page_size

    @staticmethod
    def workspace_bytes(batch: int, q_len: int, num_heads: int, max_pages: int, budget_pages: int, num_ctas: int) -> int:
        """Bytes of workspace for steps of ``batch`` requests whose block tables have ``max_pages`` entries, on a grid of ``num_ctas`` (the SM count)."""
        rows = batch * q_len
        return _aligned(_cabi.workspace_bytes(rows, 1, num_heads, num_ctas)) + _selection_bytes(rows, max_pages, budget_pages)

    @api_logged
    def run(self, q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
            softmax_scale: float, output_scale: float = 1.0, out: Optional[torch.Tensor] = None, kv_cache_sf: Optional[torch.Tensor] = None,
            summary: Optional[torch.Tensor] = None, summary_sf: Optional[torch.Tensor] = None, return_lse: bool = False,
            lse_out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """One sparse decode step on the current stream; asynchronous, capturable.  The arguments are those of the dense wrapper's ``run``
        and the summaries of the pages (``summarize_pages``); ``q`` [batch, q_len, H, 576] needs stride(0) = q_len * stride(1) when q_len > 1,
        ``kv_cache`` is 3-D and ``seq_lens`` int32.  Every query position selects for itself.  ``out`` and the base-2 LSE (of the pages that
        were attended to) are as there."""
        if self._pages is None:
            raise RuntimeError("Call plan() before run().")
        sp, dense = self._pages, self._dense
        done = _native.sparse_decode(self._workspace_buffer, dense._status, self._num_heads, self._page_size, dense._out_code, dense._num_ctas,
                                     dense._enable_pdl, dense._soft_cap, dense._sink, dense._wait_polls, sp.budget_pages, sp.sink_pages, sp.local_pages,
                                     sp.causal, q, kv_cache, block_tables, seq_lens, max_seq_len, softmax_scale, output_scale, out, kv_cache_sf,
                                     summary, summary_sf, return_lse, lse_out)
        if done is not None:
            return done
        if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[2] != self._num_heads or q.shape[3] != HEAD_DIM_QK:
            raise ValueError(f"q must have shape [batch, q_len, {self._num_heads}, {HEAD_DIM_QK}]")
        if q.device != self._device:
            raise ValueError("q must live on the device of the workspace buffer")
        batch, q_len, heads, _ = q.shape
        if q_len > 1 and batch > 1 and q.stride(0) != q_len * q.stride(1):
            raise ValueError("with several query positions stride(0) of q must be q_len * stride(1)")
        if kv_cache_sf is None or summary is None or summary_sf is None:
            raise ValueError("sparse FP4 MLA requires kv_cache_sf, summary and summary_sf")
        pages, page_size = check_cache(kv_cache, kv_cache_sf)
        if page_size != self._page_size:
            raise ValueError(f"kv_cache page size {page_size} does not match planned {self._page_size}")
        if kv_cache.device != self._device:
            raise ValueError("q, kv_cache, and kv_cache_sf must share a device")
        check_summary(summary, summary_sf, pages, self._device)
        check_tables(block_tables, seq_lens, self._device, batch)
        width = block_tables.shape[1]
        if max_seq_len <= 0 or max_seq_len > width * page_size:
            raise ValueError(f"max_seq_len must be positive and within what block_tables can address ({width} pages of {page_size} tokens), got {max_seq_len}")
        shape = (batch, q_len, heads, self._dense._kv_lora_rank)
        if out is not None and (tuple(out.shape) != shape or not out.is_contiguous()):
            raise ValueError("out must be a contiguous [batch, q_len, num_heads, 512] tensor")
        if lse_out is not None and (tuple(lse_out.shape) != shape[:3] or not lse_out.is_contiguous()):
            raise ValueError("lse_out must be a contiguous float32 [batch, q_len, num_heads] tensor on the device of q")
        if os.environ.get("MLA_FP4_VALIDATE", "0") not in ("", "0"):
            validate_page_ids(block_tables, seq_lens, page_size, pages)
        rows = batch * q_len
        selected, selected_lens, scores = self._scratch(rows, width)
        select_pages(q, summary, summary_sf, block_tables, seq_lens, page_size, sp.budget_pages, sink_pages=sp.sink_pages,
                     local_pages=sp.local_pages, causal=sp.causal, selected=selected, selected_lens=selected_lens, workspace=scores, status=dense._status)
        got = self._dense.run(q.as_strided((rows, 1, heads, HEAD_DIM_QK), (q.stride(0) if q_len == 1 else q.stride(1), 16, q.stride(2), 1)), kv_cache,
                              selected, selected_lens, min(max_seq_len, sp.budget_pages * page_size), softmax_scale, output_scale,
                              out=None if out is None else out.view(rows, 1, heads, -1), kv_cache_sf=kv_cache_sf, return_lse=return_lse,
                              lse_out=None if lse_out is None else lse_out.view(rows, 1, heads))
        if not return_lse:
            return out if out is not None else got.view(shape)
        return (out if out is not None else got[0].view(shape)), (lse_out if lse_out is not None else got[1].view(shape[:3]))

    def _scratch(self, rows: int, width: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The selection's table, lengths and scores in the workspace, behind the decode step's scratch."""
        budget = self._pages.budget_pages
        at = _aligned(_cabi.workspace_bytes(max(rows, 1), 1, self._num_heads, self._dense._num_ctas))
        need = at + _selection_bytes(rows, width, budget)
        if self._workspace_buffer.numel() < need:
            raise ValueError(f"workspace_buffer has {self._workspace_buffer.numel()} bytes, but {need} are required")
        table_end = at + 4 * rows * budget
        lens_end = table_end + 4 * rows
        scores = _aligned(lens_end)
        part = self._workspace_buffer[at:lens_end].view(torch.int32)
        return part[:rows * budget].view(rows, budget), part[rows * budget:], self._workspace_buffer[scores:need]

    @property
    def status(self) -> Optional[torch.Tensor]:
        """The device status words (int32 [8]), for ``summarize_new_pages`` to report in too."""
        return self._dense._status

    def device_status(self) -> Tuple[int, ...]:
        return self._dense.device_status()

    def check_device_status(self) -> None:
        self._dense.check_device_status()


def _aligned(n: int) -> int:
    return (n + 255) // 256 * 256


def _selection_bytes(rows: int, width: int, budget: int) -> int:
    return _aligned(4 * rows * budget + 4 * rows) + (_cabi.select_workspace_bytes(rows, 1, width) if width > budget else 0)


__all__ = ["BatchMLASparseDecodeFP4Wrapper", "SparsePages", "select_pages", "summarize_new_pages", "summarize_pages"]
