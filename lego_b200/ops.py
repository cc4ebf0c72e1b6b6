"""Kernel-level callables: the Python side of the C ABI.

The names and argument meaning follow the callables the reference generates:
``matmul(a, b, activation="")`` (``triton_generated/matmul/matmul_NTA_NTB.py:129-145``),
``softmax(x)`` (``triton_generated/softmax/softmax.py:97-160``),
``LEGOLayerNorm.apply(x, normalized_shape, weight, bias, eps)``
(``triton_generated/layernorm/layernorm.py:279-340``),
``lego_group_gemm_fn(group_A, group_B)``
(``triton_generated/grouped_gemm/grouped_gemm.py:120-162``), plus ``permute`` /
``transpose`` for the MLIR transpose programs and the index-map evaluator.  ``rotary``,
``attention`` and ``tree_attention`` (no counterpart there) are the rest of a language model's
attention layer, in training and over a paged cache.

Tensors are torch tensors; torch only owns memory and streams here.  A CUDA
tensor is processed in place on the current stream.  A CPU tensor is staged
through the device (large ones in row blocks, so that copy-in, kernel and copy-out
overlap) and a CPU tensor comes back: that is the end-to-end path.  Without a GPU or without the built library every
op raises; there is no CPU implementation behind them.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import List, Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _abi
from .layout import Col, GroupBy, OrderBy, Row
from .lowering import lower, lower_optional

__all__ = [
    "eval_apply", "eval_inv", "eval_range", "permute", "permute_plan", "permute_dma_plan", "permute_slabs", "permute_slab_info", "transpose", "softmax",
    "LEGOLayerNorm", "lego_layer_norm", "layer_norm_fwd", "layer_norm_bwd", "matmul", "lego_group_gemm_fn",
    "rotary", "rotary_frequencies", "LEGORotary", "attention", "attention_fwd", "attention_bwd", "LEGOAttention", "tree_attention",
    "grouped_swizzle_layout", "default_group_m", "default_tile_order", "row_tiling_layout", "device_status", "tune", "selftest_bounded_wait",
]


def _device() -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("lego_b200 needs a CUDA device (B200, sm_100a); there is no CPU path")
    return torch.device("cuda", torch.cuda.current_device())


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _stream_on(dev: torch.device) -> int:
    """``_stream()`` of a device by its number, without making a Stream object for it."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _to_device(t: torch.Tensor) -> torch.Tensor:
    if t.is_cuda:
        return t
    return t.to(_device(), non_blocking=True)


def _to_host(result: torch.Tensor) -> torch.Tensor:
    """A device result as a pinned host tensor (synchronises the current stream)."""
    out = torch.empty(result.shape, dtype=result.dtype, device="cpu", pin_memory=True)
    out.copy_(result, non_blocking=True)
    torch.cuda.current_stream().synchronize()
    return out


def _like_input(result: torch.Tensor, ref: torch.Tensor) -> torch.Tensor:
    """Results follow the residence of the input: CPU in, CPU out."""
    return result if ref.is_cuda else _to_host(result)


# Host-resident operands.  A host tensor is staged through the device in row blocks on
# three streams: block i + 1 is copied in while block i is computed and block i - 1 is
# copied out, so that a call on host buffers costs about one PCIe direction's time, not
# the sum of both.  Pinned inputs overlap; pageable ones still work, serialised by the
# driver's own staging.
_HOST_BLOCK_BYTES = 16 << 20   # measured best on PCIe 5 x16 (8 and 32 MiB are within 4 %)
_side_streams = {}


def _copy_streams(dev: torch.device):
    key = (dev.index, torch.cuda.current_stream().cuda_stream)
    if key not in _side_streams:
        _side_streams[key] = (torch.cuda.Stream(dev), torch.cuda.Stream(dev))
    return _side_streams[key]


class _HostPipeline:
    """Copy-in / compute / copy-out over row blocks.  ``feed(dst, src)`` copies a host
    block to the device on the inbound stream, ``ready()`` makes the compute stream wait
    for everything fed so far, ``drain(dst, src)`` sends a device block back once the
    compute stream has reached this point, ``finish()`` waits for the last block."""

    def __init__(self):
        self.dev = _device()
        self.main = torch.cuda.current_stream()
        self.inbound, self.outbound = _copy_streams(self.dev)
        self.inbound.wait_stream(self.main)
        self.outbound.wait_stream(self.main)

    def feed(self, dst: torch.Tensor, src: torch.Tensor) -> None:
        with torch.cuda.stream(self.inbound):
            dst.copy_(src, non_blocking=True)

    def ready(self) -> None:
        ev = torch.cuda.Event()
        ev.record(self.inbound)
        self.main.wait_event(ev)

    def drain(self, dst: torch.Tensor, src: torch.Tensor) -> None:
        ev = torch.cuda.Event()
        ev.record(self.main)
        self.outbound.wait_event(ev)
        with torch.cuda.stream(self.outbound):
            dst.copy_(src, non_blocking=True)

    def finish(self) -> None:
        # device blocks were allocated on the compute stream: order their reuse after both copy streams
        self.main.wait_stream(self.inbound)
        self.main.wait_stream(self.outbound)
        self.outbound.synchronize()


def _row_blocks(rows: int, row_bytes: int, multiple: int = 1):
    """Consecutive row ranges of about ``_HOST_BLOCK_BYTES`` each (whole multiples of ``multiple``
    rows except the last).  Blocks of equal size: starting and ending a long input with blocks of
    an eighth, a quarter and a half of the size -- to shorten the first copy-in and the last
    copy-out, the only transfers nothing overlaps -- measured no gain (softmax 16384 x 8192 from
    pinned memory 6.15 against 6.08 ms): a copy of 2 MiB runs at 20 GB/s, one of 4 MiB at 29,
    so the small blocks give back what they save."""
    step = max(1, _HOST_BLOCK_BYTES // max(1, row_bytes))
    step = max(multiple, step // multiple * multiple)
    return [(r0, min(rows, r0 + step)) for r0 in range(0, rows, step)]


def _pinned_like(shape, dtype) -> torch.Tensor:
    return torch.empty(tuple(shape), dtype=dtype, device="cpu", pin_memory=True)


def device_status() -> int:
    """Synchronise the current stream and return the device status word's verdict;
    raises if a bounded wait inside a kernel ran out."""
    detail = C.c_uint32(0)
    st = _abi.lib().lego_device_status(_stream(), C.byref(detail))
    if st != 0:
        for ws in _gemm_workspaces.values():   # a kernel that gave up may have left split-K flags set
            ws[:8192].zero_()
        raise _abi.LegoError(st, f"device status word 0x{detail.value:x}")
    return 0


def selftest_bounded_wait(limit_cycles: int = 1_000_000) -> None:
    """Launch the one-CTA kernel whose wait nothing completes: it gives up after
    ``limit_cycles`` SM cycles and records its code; ``device_status()`` then raises once."""
    _device()
    _abi.check(_abi.lib().lego_selftest_bounded_wait(int(limit_cycles), _stream()), "lego_selftest_bounded_wait")


def tune(gemm_blocks: Optional[int] = None, gemm_streamk: Optional[bool] = None,
         gemm_lag: Optional[int] = None, permute_dma_tile: Optional[int] = None,
         permute_dma_ctas: Optional[int] = None, permute_tile_vecs: Optional[int] = None,
         pdl_last_wave: Optional[int] = None, permute_dma_long: Optional[int] = None,
         lnbwd_min_rows: Optional[int] = None, lnbwd_fold_warp: Optional[int] = None) -> None:
    """Process-wide knobs.  GEMM: ``gemm_blocks`` 0 library's choice / 1 (256 x 256 per SM
    pair) / 2 (512 x 256 per SM pair); ``gemm_streamk`` 0 / False keeps every tile whole,
    1 / True splits a poorly filled last wave along K, 2 splits any partial wave;
    ``gemm_lag`` 0..4, the lead of the first accumulator block of a 512 x 256 tile.
    Permute: ``permute_dma_tile`` most bytes per box of the DMA kernel (0: the chunk-tiled
    kernel takes those layouts), ``permute_dma_ctas`` its CTAs per SM, ``permute_tile_vecs``
    most 16-byte vectors per tile of the chunk-tiled kernel, ``permute_dma_long`` 0: pairs whose
    common run is a whole line or more stay with the vector copy.  ``pdl_last_wave`` 1: only the last
    wave of an index-map grid lets the next grid of the stream become resident.
    ``lnbwd_min_rows``: fewest rows for which LayerNorm backward uses its ring-fed kernels
    (default 1; below, the kernel that holds a row in registers); ``lnbwd_fold_warp``: most
    consumer groups for which its grouped kernel runs a folding warp per group (0 .. 3, default 3)."""
    lib = _abi.lib()
    if lnbwd_fold_warp is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_LNBWD_FOLD_WARP, int(lnbwd_fold_warp)), "lego_tune")
    if lnbwd_min_rows is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_LNBWD_MIN_ROWS, int(lnbwd_min_rows)), "lego_tune")
    if permute_dma_tile is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_PERMUTE_DMA_TILE, int(permute_dma_tile)), "lego_tune")
    if permute_dma_ctas is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_PERMUTE_DMA_CTAS, int(permute_dma_ctas)), "lego_tune")
    if permute_tile_vecs is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_PERMUTE_TILE_VECS, int(permute_tile_vecs)), "lego_tune")
    if permute_dma_long is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_PERMUTE_DMA_LONG, int(permute_dma_long)), "lego_tune")
    if pdl_last_wave is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_PDL_LAST_WAVE, int(pdl_last_wave)), "lego_tune")
    if gemm_blocks is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_GEMM_BLOCKS, int(gemm_blocks)), "lego_tune")
    if gemm_streamk is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_GEMM_STREAMK, int(gemm_streamk)), "lego_tune")
    if gemm_lag is not None:
        _abi.check(lib.lego_tune(_abi.TUNE_GEMM_LAG, int(gemm_lag)), "lego_tune")


# One split-K scratch buffer per (device, stream): calls on one stream are ordered, calls on
# different streams must not share a buffer.  Flags (first 8 KiB) start at zero and every
# completed call leaves them zero.
_gemm_workspaces = {}


def _gemm_workspace(dev: torch.device) -> torch.Tensor:
    key = (dev.index, torch.cuda.current_stream().cuda_stream)
    ws = _gemm_workspaces.get(key)
    if ws is None:
        nbytes = _abi.lib().lego_gemm_workspace_bytes()
        if nbytes <= 0:
            raise RuntimeError("lego_gemm_workspace_bytes failed")
        if torch.cuda.is_current_stream_capturing():
            # memory allocated while capturing belongs to the graph: use it for this call only
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            ws[:8192].zero_()
            return ws
        ws = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
        _gemm_workspaces[key] = ws
    return ws


# ---- layouts used by the ops --------------------------------------------------------

def grouped_swizzle_layout(num_pid_m: int, num_pid_n: int, group_m: int = 8) -> GroupBy:
    """Tile order of the reference GEMM (``benchmarks/triton/matmul_sympy.py:57-65``):
    ``inv(pid)`` gives ``(pid_m, pid_n)`` walking ``group_m`` tile rows at a time."""
    return OrderBy(Col(max(num_pid_m // group_m, 1), 1),
                   Col(min(num_pid_m, group_m), num_pid_n)).TileBy([num_pid_m, num_pid_n])


def row_tiling_layout(n_rows: int, rows_per_tile: int = 1) -> GroupBy:
    """1-D tiling of rows, ``OrderBy(Row(n_rows)).TileBy([n_rows / R], [R])``."""
    if rows_per_tile <= 1 or n_rows % rows_per_tile:
        return OrderBy(Row(n_rows)).TileBy([n_rows])
    return OrderBy(Row(n_rows)).TileBy([n_rows // rows_per_tile], [rows_per_tile])


# ---- index-map evaluator ------------------------------------------------------------

def eval_apply(layout: GroupBy, idx: torch.Tensor) -> torch.Tensor:
    """``layout.apply`` over rows of ``idx`` (int64 ``[n, rank]``) -> int64 ``[n]``."""
    desc = lower(layout)
    if idx.dtype != torch.int64 or idx.dim() != 2 or idx.shape[1] != desc.rank:
        raise ValueError(f"idx must be int64 [n, {desc.rank}]")
    d = _to_device(idx).contiguous()
    out = torch.empty(d.shape[0], dtype=torch.int64, device=d.device)
    _abi.check(_abi.lib().lego_eval_apply(C.byref(desc), d.data_ptr(), out.data_ptr(), d.shape[0], _stream()),
               "lego_eval_apply")
    return _like_input(out, idx)


def eval_inv(layout: GroupBy, flat: torch.Tensor) -> torch.Tensor:
    """``layout.inv`` over ``flat`` (int64 ``[n]``) -> int64 ``[n, rank]``."""
    desc = lower(layout)
    if flat.dtype != torch.int64 or flat.dim() != 1:
        raise ValueError("flat must be int64 [n]")
    d = _to_device(flat).contiguous()
    out = torch.empty((d.shape[0], desc.rank), dtype=torch.int64, device=d.device)
    _abi.check(_abi.lib().lego_eval_inv(C.byref(desc), d.data_ptr(), out.data_ptr(), d.shape[0], _stream()),
               "lego_eval_inv")
    return _like_input(out, flat)


def eval_range(layout: GroupBy, begin: int = 0, count: Optional[int] = None, host: bool = False) -> torch.Tensor:
    """``layout.apply`` over logical flat ids ``begin .. begin+count`` -> int64, on the
    device, or with ``host=True`` in pinned host memory (evaluated block by block, each
    block leaving the device while the next is computed)."""
    desc = lower(layout)
    size = layout.size()
    if count is None:
        count = size - begin
    call = _abi.lib().lego_eval_range
    if host and count * 8 > 2 * _HOST_BLOCK_BYTES:
        pipe = _HostPipeline()
        res = _pinned_like((count,), torch.int64)
        bufs = [torch.empty(_HOST_BLOCK_BYTES // 8, dtype=torch.int64, device=pipe.dev) for _ in range(2)]
        done = [None, None]  # the copy-out that last read each buffer
        for i, (r0, r1) in enumerate(_row_blocks(count, 8)):
            buf = bufs[i & 1][: r1 - r0]
            if done[i & 1] is not None:
                pipe.main.wait_event(done[i & 1])
            _abi.check(call(C.byref(desc), begin + r0, r1 - r0, buf.data_ptr(), _stream()), "lego_eval_range")
            pipe.drain(res[r0:r1], buf)
            done[i & 1] = torch.cuda.Event()
            done[i & 1].record(pipe.outbound)
        pipe.finish()
        return res
    out = torch.empty(count, dtype=torch.int64, device=_device())
    _abi.check(call(C.byref(desc), begin, count, out.data_ptr(), _stream()), "lego_eval_range")
    return _to_host(out) if host else out


# ---- layout reorganisation ----------------------------------------------------------

def permute_plan(elem_bytes: int, src: GroupBy, dst: GroupBy, tile_order: Optional[GroupBy] = None):
    """Which kernel ``permute`` would run: ``(kind, tile_in, tile_out)`` with kind
    0 staged, 1 gather, 2 shared-memory tiled transpose, 3 TMA-fed tiled transpose,
    4 chunk-tiled permute, 5 DMA permute.  Host-only; needs no GPU."""
    kind, ti, to = C.c_int32(0), C.c_int64(0), C.c_int64(0)
    _abi.check(_abi.lib().lego_permute_plan(elem_bytes, C.byref(lower(src)), C.byref(lower(dst)),
                                            lower_optional(tile_order), C.byref(kind), C.byref(ti), C.byref(to)),
               "lego_permute_plan")
    return kind.value, ti.value, to.value


def permute_dma_plan(elem_bytes: int, src: GroupBy, dst: GroupBy, slabs: int = -1) -> dict:
    """The DMA permute's plan for a pair of layouts: both tensor maps (``size``, ``stride``,
    ``box`` per dimension, innermost first, in elements of ``elem_bytes``) and the digits of
    the tile id; ``slabs >= 0``: the plan of that many slabs (``permute_slabs``).  Raises
    ``ValueError`` when the pair is not moved that way.  Host-only."""
    plan = _abi.DmaPlan()
    _abi.check(_abi.lib().lego_permute_dma_plan(elem_bytes, C.byref(lower(src)), C.byref(lower(dst)), int(slabs),
                                                C.byref(plan)), "lego_permute_dma_plan")

    def side(sd):
        return {k: [int(getattr(sd, k)[i]) for i in range(sd.rank)] for k in ("size", "stride", "box")}

    return {"elem_bytes": plan.elem_bytes, "n_tiles": plan.n_tiles, "tile_bytes": plan.tile_bytes,
            "load": side(plan.load), "store": side(plan.store),
            "outer": [{"radix": int(o.radix), "ld": (o.ld_dim, o.ld_mul), "st": (o.st_dim, o.st_mul)}
                      for o in plan.outer[:plan.n_outer]]}


def permute_slab_info(elem_bytes: int, src: GroupBy, dst: GroupBy):
    """``(n_slabs, slab_elems)`` when the slowest digit of the flat index is the same logical
    digit in both layouts -- the re-layout then is ``n_slabs`` independent pieces, each
    contiguous in both buffers -- else ``None``.  Host-only."""
    n, e = C.c_int64(0), C.c_int64(0)
    st = _abi.lib().lego_permute_slab_info(elem_bytes, C.byref(lower(src)), C.byref(lower(dst)), C.byref(n),
                                           C.byref(e))
    if st == _abi.ERR_UNSUPPORTED:
        return None
    _abi.check(st, "lego_permute_slab_info")
    return n.value, e.value


def permute_slabs(x: torch.Tensor, src: GroupBy, dst: GroupBy, count: int,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The re-layout ``src -> dst`` restricted to ``count`` consecutive slabs (see
    ``permute_slab_info``): ``x`` and the result hold those slabs only."""
    d = _to_device(x).contiguous()
    res = out if out is not None else torch.empty_like(d)
    if not res.is_cuda or not res.is_contiguous() or res.numel() != d.numel() or res.dtype != d.dtype:
        raise ValueError("out must be a contiguous CUDA tensor of x's size and dtype")
    info = permute_slab_info(d.element_size(), src, dst)
    if info is None:
        raise ValueError("this pair of layouts does not split into slabs")
    if count < 0 or count > info[0] or d.numel() != count * info[1]:
        raise ValueError(f"{count} slabs of {info[1]} elements do not match a tensor of {d.numel()}")
    _abi.check(_abi.lib().lego_permute_slabs(d.data_ptr(), res.data_ptr(), d.element_size(), C.byref(lower(src)),
                                             C.byref(lower(dst)), int(count), _stream()), "lego_permute_slabs")
    return _like_input(res, x)


def _permute_from_host(x, src, dst, n_slabs, slab_elems):
    """A re-layout that splits into slabs, on a host buffer: groups of slabs of about 16 MiB go
    through the device on three streams (copy in / move / copy out), so the call costs about
    one PCIe direction instead of copy-in + kernel + copy-out."""
    eb = x.element_size()
    pipe = _HostPipeline()
    lib = _abi.lib()
    flat = x.reshape(-1)
    out = _pinned_like((x.numel(),), x.dtype)
    d_in = torch.empty(x.numel(), dtype=x.dtype, device=pipe.dev)
    d_out = torch.empty_like(d_in)
    s_desc, d_desc = lower(src), lower(dst)
    for k0, k1 in _row_blocks(n_slabs, slab_elems * eb):
        e0, e1 = k0 * slab_elems, k1 * slab_elems
        pipe.feed(d_in[e0:e1], flat[e0:e1])
        pipe.ready()
        _abi.check(lib.lego_permute_slabs(d_in[e0:e1].data_ptr(), d_out[e0:e1].data_ptr(), eb, C.byref(s_desc),
                                          C.byref(d_desc), k1 - k0, _stream()), "lego_permute_slabs")
        pipe.drain(out[e0:e1], d_out[e0:e1])
    pipe.finish()
    return out.reshape(x.shape)


def permute(x: torch.Tensor, src: GroupBy, dst: GroupBy, tile_order: Optional[GroupBy] = None,
            out: Optional[torch.Tensor] = None, tiles: Optional[Sequence[int]] = None) -> torch.Tensor:
    """``out_flat[dst(idx)] = x_flat[src(idx)]`` over the layouts' common logical
    domain.  ``x`` is read as a flat contiguous buffer; the result has x's shape.
    ``tiles=(begin, count)`` moves only that range of ``tile_order`` ids (one GPU's
    slab of a reorganisation split across several) and leaves the rest of ``out`` alone."""
    if src.size() != x.numel():
        raise ValueError(f"layout covers {src.size()} elements, tensor has {x.numel()}")
    if (not x.is_cuda and out is None and tiles is None and tile_order is None and x.is_contiguous()
            and x.numel() * x.element_size() > 2 * _HOST_BLOCK_BYTES):
        info = permute_slab_info(x.element_size(), src, dst)
        if info is not None and info[0] * info[1] == x.numel() and info[1] * x.element_size() <= _HOST_BLOCK_BYTES:
            return _permute_from_host(x, src, dst, *info)
    d = _to_device(x).contiguous()
    res = out if out is not None else torch.empty_like(d)
    if not res.is_cuda or not res.is_contiguous() or res.numel() != d.numel() or res.dtype != d.dtype:
        raise ValueError("out must be a contiguous CUDA tensor of x's size and dtype")
    if tiles is not None:
        begin, count = tiles
        _abi.check(_abi.lib().lego_permute_tiles(d.data_ptr(), res.data_ptr(), d.element_size(), C.byref(lower(src)),
                                                 C.byref(lower(dst)), lower_optional(tile_order), int(begin),
                                                 int(count), _stream()), "lego_permute_tiles")
        return _like_input(res, x)
    _abi.check(_abi.lib().lego_permute(d.data_ptr(), res.data_ptr(), d.element_size(), C.byref(lower(src)),
                                       C.byref(lower(dst)), lower_optional(tile_order), _stream()),
               "lego_permute")
    return _like_input(res, x)


def transpose(x: torch.Tensor, tile: int = 32, tile_order: Optional[GroupBy] = None) -> torch.Tensor:
    """2-D transpose through the tiled layouts of the reference's MLIR programs
    (``benchmarks/mlir/transpose_smem.py:33-37``): source viewed row-major in
    ``tile x tile`` tiles, destination column-major, tiles visited in ``tile_order``
    (default: column-major over tiles)."""
    if x.dim() != 2:
        raise ValueError("transpose expects a matrix")
    r, c = x.shape
    if r % tile or c % tile:
        raise ValueError(f"matrix {r}x{c} is not a multiple of the {tile}x{tile} tile")
    src = OrderBy(Row(r, c)).TileBy([r // tile, c // tile], [tile, tile])
    dst = OrderBy(Col(r, c)).TileBy([r // tile, c // tile], [tile, tile])
    default_order = tile_order is None
    if default_order:
        tile_order = OrderBy(Col(r // tile, c // tile)).TileBy([r // tile, c // tile])
    nbytes = x.numel() * x.element_size()
    if (not x.is_cuda and x.is_contiguous() and default_order and nbytes > 2 * _HOST_BLOCK_BYTES
            and permute_plan(x.element_size(), src, dst, tile_order)[0] in (2, 3)):
        return _transpose_from_host(x, tile, src, dst, tile_order)
    return permute(x, src, dst, tile_order).reshape(c, r)


def _transpose_from_host(x, tile, src, dst, tile_order):
    """Host matrix: slabs of output rows.  A slab's input is a band of columns, copied in with
    one strided copy; its tiles are a contiguous range of the column-major tile order; its
    output rows are contiguous.  Slab i + 1 arrives while slab i is transposed and slab i - 1
    leaves, so the call costs about one PCIe direction instead of copy-in + kernel + copy-out."""
    r, c = x.shape
    eb = x.element_size()
    pipe = _HostPipeline()
    lib = _abi.lib()
    d_in = torch.empty((r, c), dtype=x.dtype, device=pipe.dev)
    d_out = torch.empty((c, r), dtype=x.dtype, device=pipe.dev)
    out = _pinned_like((c, r), x.dtype)
    tiles_down = r // tile
    for c0, c1 in _row_blocks(c, r * eb, multiple=tile):        # bands of columns
        _abi.check(lib.lego_copy_2d(d_in.data_ptr() + c0 * eb, c * eb, x.data_ptr() + c0 * eb, c * eb,
                                    (c1 - c0) * eb, r, pipe.inbound.cuda_stream), "lego_copy_2d")
        pipe.ready()
        permute(d_in, src, dst, tile_order, out=d_out.reshape(r, c),
                tiles=(c0 // tile * tiles_down, (c1 - c0) // tile * tiles_down))
        pipe.drain(out[c0:c1], d_out[c0:c1])
    pipe.finish()
    return out


# ---- row-wise kernels ---------------------------------------------------------------

def softmax(x: torch.Tensor, row_map: Optional[GroupBy] = None) -> torch.Tensor:
    """Row-wise softmax of a 2-D fp16 or fp32 tensor (fp32 arithmetic)."""
    if x.dim() != 2:
        raise ValueError("softmax expects a 2-D tensor")
    fn = {torch.float16: "lego_softmax_f16", torch.float32: "lego_softmax_f32"}.get(x.dtype)
    if fn is None:
        raise ValueError(f"softmax supports float16 and float32, got {x.dtype}")
    call = getattr(_abi.lib(), fn)
    if not x.is_cuda and x.is_contiguous() and x.numel() * x.element_size() > 2 * _HOST_BLOCK_BYTES:
        # Host rows: staged block by block.  A row map only decides which CTA takes which
        # row, never the result, so the blocks run in arrival order without it.
        lower_optional(row_map)
        pipe = _HostPipeline()
        d = torch.empty(x.shape, dtype=x.dtype, device=pipe.dev)
        y = torch.empty_like(d)
        out = _pinned_like(x.shape, x.dtype)
        for r0, r1 in _row_blocks(x.shape[0], x.shape[1] * x.element_size()):
            pipe.feed(d[r0:r1], x[r0:r1])
            pipe.ready()
            _abi.check(call(d[r0:r1].data_ptr(), y[r0:r1].data_ptr(), r1 - r0, x.shape[1], None, _stream()), fn)
            pipe.drain(out[r0:r1], y[r0:r1])
        pipe.finish()
        return out
    d = _to_device(x).contiguous()
    y = torch.empty_like(d)
    n_rows, n_cols = d.shape
    _abi.check(call(d.data_ptr(), y.data_ptr(), n_rows, n_cols, lower_optional(row_map), _stream()), fn)
    return _like_input(y, x)


def layer_norm_fwd(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float,
                   row_map: Optional[GroupBy] = None):
    """LayerNorm forward over the last axis: ``(y, mean, rstd)``, statistics fp32."""
    if x.dtype != torch.float16 or weight.dtype != torch.float16 or bias.dtype != torch.float16:
        raise ValueError("layer norm supports float16 tensors")
    n = x.shape[-1]
    if weight.numel() != n or bias.numel() != n:
        raise ValueError("weight / bias must have the size of the last axis")
    if n * x.element_size() > 65536:
        raise RuntimeError("This layer norm doesn't support feature dim >= 64KB.")
    call = _abi.lib().lego_layernorm_fwd_f16
    if not x.is_cuda and x.is_contiguous() and x.numel() * x.element_size() > 2 * _HOST_BLOCK_BYTES:
        # host rows: staged block by block (a row map never changes the result, see softmax)
        lower_optional(row_map)
        pipe = _HostPipeline()
        xh = x.reshape(-1, n)
        m = xh.shape[0]
        w, b = _to_device(weight).contiguous(), _to_device(bias).contiguous()
        d = torch.empty(xh.shape, dtype=x.dtype, device=pipe.dev)
        y = torch.empty_like(d)
        mean = torch.empty(m, dtype=torch.float32, device=pipe.dev)
        rstd = torch.empty(m, dtype=torch.float32, device=pipe.dev)
        y_h, mean_h, rstd_h = _pinned_like(xh.shape, x.dtype), _pinned_like((m,), torch.float32), _pinned_like((m,), torch.float32)
        for r0, r1 in _row_blocks(m, n * x.element_size()):
            pipe.feed(d[r0:r1], xh[r0:r1])
            pipe.ready()
            _abi.check(call(d[r0:r1].data_ptr(), w.data_ptr(), b.data_ptr(), y[r0:r1].data_ptr(),
                            mean[r0:r1].data_ptr(), rstd[r0:r1].data_ptr(), r1 - r0, n, float(eps), None, _stream()),
                       "lego_layernorm_fwd_f16")
            pipe.drain(y_h[r0:r1], y[r0:r1])
        pipe.drain(mean_h, mean)
        pipe.drain(rstd_h, rstd)
        pipe.finish()
        return y_h.reshape(x.shape), mean_h, rstd_h
    d = _to_device(x).contiguous()
    x2 = d.reshape(-1, n)
    w, b = _to_device(weight).contiguous(), _to_device(bias).contiguous()
    m = x2.shape[0]
    y = torch.empty_like(d)
    mean = torch.empty(m, dtype=torch.float32, device=d.device)
    rstd = torch.empty(m, dtype=torch.float32, device=d.device)
    _abi.check(_abi.lib().lego_layernorm_fwd_f16(x2.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(),
                                                 mean.data_ptr(), rstd.data_ptr(), m, n, float(eps),
                                                 lower_optional(row_map), _stream()),
               "lego_layernorm_fwd_f16")
    return _like_input(y, x), _like_input(mean, x), _like_input(rstd, x)


class LEGOLayerNorm(torch.autograd.Function):
    """``LEGOLayerNorm.apply(x, normalized_shape, weight, bias, eps)``."""

    @staticmethod
    def forward(ctx, x, normalized_shape, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(dy, x, w, mean, rstd)
        return dx, None, dw, db, None


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor):
    """LayerNorm backward over the last axis: ``(dx, dweight, dbias)`` from the saved
    row statistics; dweight / dbias come from a fixed-order two-stage column reduction
    (same bits on every run)."""
    n = x.shape[-1]
    if (not x.is_cuda and not dy.is_cuda and x.is_contiguous() and dy.is_contiguous() and x.shape == dy.shape
            and x.dtype == torch.float16 and dy.dtype == torch.float16 and weight.dtype == torch.float16
            and x.numel() * 2 > 2 * _HOST_BLOCK_BYTES):
        return _layer_norm_bwd_from_host(dy, x, weight, mean, rstd)
    xd = _to_device(x).contiguous().reshape(-1, n)
    dyd = _to_device(dy).contiguous().reshape(-1, n)
    wd = _to_device(weight).contiguous()
    md, rd = _to_device(mean).contiguous(), _to_device(rstd).contiguous()
    m = xd.shape[0]
    if dyd.shape != xd.shape or wd.numel() != n or md.numel() != m or rd.numel() != m:
        raise ValueError("layer norm backward: shapes of dy, x, weight, mean, rstd do not agree")
    if xd.dtype != torch.float16 or dyd.dtype != torch.float16 or wd.dtype != torch.float16:
        raise ValueError("layer norm supports float16 tensors")
    lib = _abi.lib()
    prow = lib.lego_layernorm_bwd_partial_rows(m, n)
    partial = torch.empty((2, prow, n), dtype=torch.float32, device=xd.device)
    dx = torch.empty_like(xd)
    dw = torch.empty_like(wd)
    db = torch.empty_like(wd)
    _abi.check(lib.lego_layernorm_bwd_f16(dyd.data_ptr(), xd.data_ptr(), wd.data_ptr(), md.data_ptr(),
                                          rd.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                          partial.data_ptr(), m, n, _stream()),
               "lego_layernorm_bwd_f16")
    return _like_input(dx.reshape(x.shape), x), _like_input(dw, weight), _like_input(db, weight)


def _layer_norm_bwd_from_host(dy, x, weight, mean, rstd):
    """Host rows of x and dy: staged block by block (copy-in / compute / copy-out overlap).  Every
    block yields its own dweight / dbias (fp16, as the entry point rounds them); they are summed
    in fp32 on the device and rounded once more at the end, so these two results may differ in
    the last bit from one call on device-resident rows."""
    n = x.shape[-1]
    xh, dyh = x.reshape(-1, n), dy.reshape(-1, n)
    m = xh.shape[0]
    if weight.numel() != n or mean.numel() != m or rstd.numel() != m:
        raise ValueError("layer norm backward: shapes of dy, x, weight, mean, rstd do not agree")
    pipe = _HostPipeline()
    lib = _abi.lib()
    wd = _to_device(weight).contiguous()
    md, rd = _to_device(mean).contiguous(), _to_device(rstd).contiguous()
    xd = torch.empty(xh.shape, dtype=x.dtype, device=pipe.dev)
    dyd = torch.empty_like(xd)
    dx = torch.empty_like(xd)
    dx_h = _pinned_like(xh.shape, x.dtype)
    dw32 = torch.zeros(n, dtype=torch.float32, device=pipe.dev)
    db32 = torch.zeros(n, dtype=torch.float32, device=pipe.dev)
    dw_b, db_b = torch.empty_like(wd), torch.empty_like(wd)
    blocks = _row_blocks(m, n * 2, multiple=4)
    prow = lib.lego_layernorm_bwd_partial_rows(max(r1 - r0 for r0, r1 in blocks), n)
    partial = torch.empty((2, prow, n), dtype=torch.float32, device=pipe.dev)
    for r0, r1 in blocks:
        pipe.feed(xd[r0:r1], xh[r0:r1])
        pipe.feed(dyd[r0:r1], dyh[r0:r1])
        pipe.ready()
        _abi.check(lib.lego_layernorm_bwd_f16(dyd[r0:r1].data_ptr(), xd[r0:r1].data_ptr(), wd.data_ptr(),
                                              md[r0:r1].data_ptr(), rd[r0:r1].data_ptr(), dx[r0:r1].data_ptr(),
                                              dw_b.data_ptr(), db_b.data_ptr(), partial.data_ptr(), r1 - r0, n, _stream()),
                   "lego_layernorm_bwd_f16")
        dw32 += dw_b
        db32 += db_b
        pipe.drain(dx_h[r0:r1], dx[r0:r1])
    dw, db = dw32.to(torch.float16), db32.to(torch.float16)
    pipe.finish()
    return dx_h.reshape(x.shape), _like_input(dw, weight), _like_input(db, weight)


lego_layer_norm = LEGOLayerNorm.apply


# ---- GEMM ---------------------------------------------------------------------------

def _operand(t: torch.Tensor):
    """(contiguous storage, transposed?) of a 2-D operand that is either
    contiguous or the ``.T`` view of a contiguous matrix."""
    if t.is_contiguous():
        return t, 0
    if t.t().is_contiguous():
        return t.t(), 1
    return t.contiguous(), 0


# Rows of 128 x 256 tiles walked together by the default tile order.  One wave of the
# persistent kernel covers 74 tiles of 512 x 256: with GROUP_M tile rows per group it reads a
# GROUP_M * 128-row panel of A and 74 * 512 / (GROUP_M * 128) tile columns of B.  GROUP_M = 8
# (the value the reference tunes for its own kernel) makes a wave read every column of an
# 8192-wide B; 32 makes the wave nearly square (A panel 64 MiB + B 36 MiB for K = 8192 in
# fp16) and the A panel stays in the 126 MB L2 from wave to wave: 8192^3 fp16 sustained
# 1 224 -> 1 271 TFLOP/s on one box, DRAM reads per launch 1.17 GB -> about a third.
_A_PANEL_BYTES = 72 << 20


def default_group_m(num_pid_m: int, k: int, elem_bytes: int) -> int:
    """GROUP_M of the default tile order: the largest of 32, 16, 8 that tiles ``num_pid_m``
    and whose A panel (GROUP_M * 128 rows x K) stays within about half of L2."""
    for gm in (32, 16, 8):
        if (num_pid_m % gm == 0 or num_pid_m <= gm) and (gm == 8 or min(gm, num_pid_m) * 128 * k * elem_bytes <= _A_PANEL_BYTES):
            return gm
    return 8


def default_tile_order(m: int, n: int, k: int, elem_bytes: int = 2, group_m: Optional[int] = None) -> Optional[GroupBy]:
    """The tile order ``matmul`` uses when the caller passes none: the reference's grouped
    swizzle over the grid of 128 x 256 tiles, or None (row-major) when GROUP_M does not tile it."""
    npm, npn = -(-m // 128), -(-n // 256)
    gm = default_group_m(npm, k, elem_bytes) if group_m is None else group_m
    if npm % gm == 0 or npm <= gm:
        return grouped_swizzle_layout(npm, npn, gm)
    return None


def matmul(a: torch.Tensor, b: torch.Tensor, activation: str = "", tile_order: Optional[GroupBy] = None,
           group_m: Optional[int] = None) -> torch.Tensor:
    """``C = act(A @ B)``: fp16 in, fp32 accumulate, fp16 out.  Either operand may
    be a ``.T`` view.  Tile order defaults to the reference's grouped swizzle with
    ``GROUP_M = group_m`` (chosen by ``default_group_m`` when None) when it is a bijection
    for the tile grid, row-major otherwise."""
    if a.dtype != b.dtype or a.dtype not in (torch.float16, torch.float8_e5m2):
        raise ValueError("matmul supports float16 operands, or float8_e5m2 operands (fp16 result)")
    fn = "lego_gemm_f16" if a.dtype == torch.float16 else "lego_gemm_e5m2"
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError("Incompatible dimensions")
    act = {"": _abi.ACT_NONE, "leaky_relu": _abi.ACT_LEAKY_RELU}.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}")
    m, k = a.shape
    n = b.shape[1]
    lib = _abi.lib()
    if (not a.is_cuda and not b.is_cuda and a.is_contiguous() and tile_order is None
            and a.numel() * a.element_size() > 2 * _HOST_BLOCK_BYTES and m % 256 == 0):
        # Host operands: B goes in first, then A in blocks of rows; each block's rows of C
        # leave while the next block arrives.  Every block is its own GEMM with its own
        # default tile order.
        pipe = _HostPipeline()
        if not b.is_contiguous() and b.t().is_contiguous():  # a .T view: copy the storage, keep the view
            store = torch.empty(b.t().shape, dtype=b.dtype, device=pipe.dev)
            pipe.feed(store, b.t())
            bd = store.t()
        else:
            bd = torch.empty(b.shape, dtype=b.dtype, device=pipe.dev)
            pipe.feed(bd, b)
        b_st, tb = _operand(bd)
        ad = torch.empty(a.shape, dtype=a.dtype, device=pipe.dev)
        c = torch.empty((m, n), dtype=torch.float16, device=pipe.dev)
        c_h = _pinned_like((m, n), torch.float16)
        call = getattr(lib, fn + "_ws")
        ws = _gemm_workspace(pipe.dev)
        for r0, r1 in _row_blocks(m, max(k * a.element_size(), n * 2), multiple=256):
            pipe.feed(ad[r0:r1], a[r0:r1])
            pipe.ready()
            order = default_tile_order(r1 - r0, n, k, a.element_size(), group_m)
            _abi.check(call(ad[r0:r1].data_ptr(), b_st.data_ptr(), c[r0:r1].data_ptr(), r1 - r0, n, k,
                            0, tb, act, lower_optional(order), ws.data_ptr(), ws.numel(), _stream()), fn)
            pipe.drain(c_h[r0:r1], c[r0:r1])
        pipe.finish()
        return c_h
    ad, bd = _to_device(a), _to_device(b)
    a_st, ta = _operand(ad)
    b_st, tb = _operand(bd)
    c = torch.empty((m, n), dtype=torch.float16, device=ad.device)
    if tile_order is None:
        tile_order = default_tile_order(m, n, k, a.element_size(), group_m)
    ws = _gemm_workspace(ad.device)
    _abi.check(getattr(lib, fn + "_ws")(a_st.data_ptr(), b_st.data_ptr(), c.data_ptr(), m, n, k, ta, tb, act,
                                        lower_optional(tile_order), ws.data_ptr(), ws.numel(), _stream()), fn)
    return _like_input(c, a)


def lego_group_gemm_fn(group_A: Sequence[torch.Tensor], group_B: Sequence[torch.Tensor],
                       tile_orders: Optional[Sequence[Optional[GroupBy]]] = None) -> List[torch.Tensor]:
    """Grouped GEMM: ``[A_g @ B_g for g]`` in one persistent launch."""
    assert len(group_A) == len(group_B)
    g = len(group_A)
    if g == 0:
        return []
    if g > _abi.MAX_GROUPS:
        raise ValueError(f"at most {_abi.MAX_GROUPS} groups per call")
    for A, B in zip(group_A, group_B):
        if A.dtype != torch.float16 or B.dtype != torch.float16:
            raise ValueError("grouped GEMM supports float16 operands")
        assert A.shape[1] == B.shape[0]
    if all(not t.is_cuda for t in list(group_A) + list(group_B)) and g > 1:
        return _group_gemm_from_host(group_A, group_B, tile_orders)
    a_dev, b_dev, c_dev, mnk = [], [], [], []
    for A, B in zip(group_A, group_B):
        ad, bd = _to_device(A).contiguous(), _to_device(B).contiguous()
        a_dev.append(ad)
        b_dev.append(bd)
        c_dev.append(torch.empty((A.shape[0], B.shape[1]), dtype=torch.float16, device=ad.device))
        mnk += [A.shape[0], B.shape[1], A.shape[1]]
    PtrArr = C.c_void_p * g
    ap = PtrArr(*[t.data_ptr() for t in a_dev])
    bp = PtrArr(*[t.data_ptr() for t in b_dev])
    cp = PtrArr(*[t.data_ptr() for t in c_dev])
    sizes = (C.c_int64 * (3 * g))(*mnk)
    orders = None
    if tile_orders is not None:
        keep = [None if o is None else lower(o) for o in tile_orders]
        orders = (_abi.LayoutP * g)(*[C.cast(None, _abi.LayoutP) if o is None else C.pointer(o) for o in keep])
    _abi.check(_abi.lib().lego_grouped_gemm_f16(ap, bp, cp, sizes, g, orders, _stream()),
               "lego_grouped_gemm_f16")
    return [_like_input(c, A) for c, A in zip(c_dev, group_A)]


def _group_gemm_from_host(group_A, group_B, tile_orders) -> List[torch.Tensor]:
    """Grouped GEMM on host operands: group g + 1 is copied in while group g is computed
    (one single-problem launch each) and group g - 1 is copied out."""
    pipe = _HostPipeline()
    lib = _abi.lib()
    outs, keep = [], []
    for i, (A, B) in enumerate(zip(group_A, group_B)):
        ad = torch.empty(A.shape, dtype=A.dtype, device=pipe.dev)
        bd = torch.empty(B.shape, dtype=B.dtype, device=pipe.dev)
        cd = torch.empty((A.shape[0], B.shape[1]), dtype=torch.float16, device=pipe.dev)
        keep += [ad, bd, cd]
        pipe.feed(ad, A)
        pipe.feed(bd, B)
        pipe.ready()
        order = None if tile_orders is None or tile_orders[i] is None else lower(tile_orders[i])
        orders = None if order is None else (_abi.LayoutP * 1)(C.pointer(order))
        _abi.check(lib.lego_grouped_gemm_f16((C.c_void_p * 1)(ad.data_ptr()), (C.c_void_p * 1)(bd.data_ptr()),
                                             (C.c_void_p * 1)(cd.data_ptr()),
                                             (C.c_int64 * 3)(A.shape[0], B.shape[1], A.shape[1]), 1, orders, _stream()),
                   "lego_grouped_gemm_f16")
        out = _pinned_like(cd.shape, torch.float16)
        pipe.drain(out, cd)
        outs.append(out)
    pipe.finish()
    return outs


# ---- attention ----------------------------------------------------------------------

_ATTN_TYPES = {torch.float16: _abi.F16, torch.bfloat16: _abi.BF16}
_ROTARY_TYPES = {**_ATTN_TYPES, torch.float32: _abi.F32}


def _same_device(*tensors: Optional[torch.Tensor]) -> torch.device:
    """The device of a call: that of its CUDA tensors, which have to share one (host tensors are
    staged to it); the current device when all are host tensors."""
    at = -1
    for t in tensors:
        if t is not None:
            n = t.get_device()
            if n != at and n >= 0:
                if at >= 0:
                    raise ValueError(f"tensors on different devices: cuda:{at} and cuda:{n}")
                at = n
    return torch.device("cuda", at) if at >= 0 else _device()


_HERE = contextlib.nullcontext()


def _on(dev: torch.device):
    """The call's device made current, where it is not."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _ready(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    return t if t.is_cuda else t.to(dev, non_blocking=True)


def _dense(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """On the device, contiguous, on a 16-byte boundary."""
    t = _ready(t, dev).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strided(t: torch.Tensor, dev: torch.device):
    """A tensor ``[a, b, c, D]`` on the device in a form the kernels read in place -- last axis
    contiguous, the other strides whole 16-byte steps, the first value on such a boundary; a copy
    where it is not -- and the strides of its leading axes in elements."""
    if not t.is_cuda:
        t = t.to(dev, non_blocking=True)
    _, b, c, d = t.shape
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, (b * c * d, c * d, d)
        steps = 16 // t.element_size()
        if t.stride(-1) == 1 and all(n == 1 or (s > 0 and s % steps == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1])):
            return t, _strides(t)
    return _dense(t, dev), (b * c * d, c * d, d)


def _rows(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """On the device, the last axis contiguous."""
    t = _ready(t, dev)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t: torch.Tensor):
    """Strides of the leading axes of ``[a, b, c, D]`` in elements; an axis of one has none of its own."""
    a, b, c, d = t.shape
    s = t.stride()
    return (s[0] if a != 1 else d, s[1] if b != 1 else d, s[2] if c != 1 else d)


def _check_int32(t: torch.Tensor, name: str, shape) -> None:
    if t.dtype != torch.int32 or t.shape != shape:
        raise ValueError(f"{name} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def _check_slopes(t: torch.Tensor, heads: int) -> None:
    if t.dtype != torch.float32 or t.shape != (heads,):
        raise ValueError(f"slopes must be float32 [{heads}], got {t.dtype} {list(t.shape)}")


def _check_tangents(*tensors) -> None:
    """Refuses dual tensors: there is no forward-mode derivative, and a result without a tangent would be one of zero."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("no forward-mode derivative is computed: take the tensors' primals")


def _check_constants(**given) -> None:
    """Refuses what takes no gradient and asks for one.  Called before an autograd function is entered:
    inside its forward pass the grad mode is off."""
    for name, t in given.items():
        if isinstance(t, torch.Tensor) and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} is a constant of the operator: no gradient is computed for it")


def _optional(t: Optional[torch.Tensor], dev: torch.device) -> Optional[torch.Tensor]:
    return None if t is None else _ready(t, dev).contiguous()


def _scores(scale: Optional[float], softcap: float, dim: int):
    scale = dim ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not math.isfinite(scale) or not math.isfinite(softcap) or softcap < 0:
        raise ValueError("scale must be finite, softcap finite and not negative")
    return scale, softcap


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 8192, low: float = 1.0, high: float = 4.0, device=None) -> torch.Tensor:
    """Angles per position of the ``dim / 2`` pairs ``rotary`` turns, float64:
    ``base ** (-2 p / dim)``, stretched for contexts ``factor`` times the trained ``original_length``
    by ``scaling``: ``"linear"`` all of them; ``"ntk"`` through the base, the first pair not at all and the
    last one fully; ``"bands"`` by how often a pair turns within the trained length: at least ``high``
    times, kept; at most ``low`` times, stretched fully; blended linearly in between."""
    if dim < 2 or dim % 2:
        raise ValueError("dim must be even and at least 2")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor >= 1):
        raise ValueError("base must be positive and factor at least 1")
    if scaling == "ntk":
        base = base * factor ** (dim / (dim - 2)) if dim > 2 else base
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        if original_length < 1 or not 0 <= low < high:
            raise ValueError("bands need original_length >= 1 and 0 <= low < high")
        keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return f if device is None else f.to(device)


def _rotary(xs, positions, freqs, pairs, scale, inverse):
    """Turned copies of ``xs`` (one or two tensors ``[B, S, H_i, D]``), one launch."""
    _check_tangents(*xs, freqs)
    kind = {"half": _abi.PAIRS_HALF, "interleaved": _abi.PAIRS_INTERLEAVED}.get(pairs)
    if kind is None:
        raise ValueError(f"pairs must be 'half' or 'interleaved', got {pairs!r}")
    x = xs[0]
    code = _ROTARY_TYPES.get(x.dtype)
    if x.dim() != 4 or code is None:
        raise ValueError("rotary takes [B, S, H, D] tensors of one type: float16, bfloat16 or float32")
    B, S, H, D = x.shape
    two = xs[1] if len(xs) > 1 else None
    H2 = 0
    if two is not None:
        if two.dim() != 4 or two.dtype != x.dtype:
            raise ValueError("rotary takes [B, S, H, D] tensors of one type: float16, bfloat16 or float32")
        B2, S2, H2, D2 = two.shape
        if B2 != B or S2 != S or D2 != D:
            raise ValueError("the tensors must agree in batch, length and head size")
    at = positions.shape
    if positions.dtype not in (torch.int32, torch.int64) or len(at) not in (1, 2) or at[-1] != S or at[0] != (B if len(at) == 2 else S):
        raise ValueError(f"positions must be int32 or int64 [{B}, {S}] or [{S}]")
    turns = freqs.numel()
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or turns < 1 or 2 * turns > D:
        raise ValueError(f"freqs must be float64 of 1 .. {D // 2} pairs")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    dev = _same_device(x, two, positions, freqs)
    with _on(dev):
        pos, fr = _ready(positions, dev), _ready(freqs, dev).contiguous()
        one, y1, ptr2, y2, st2 = _rows(x, dev), torch.empty((B, S, H, D), dtype=x.dtype, device=dev), None, None, (0, 0, 0)
        if two is not None:
            second, y2 = _rows(two, dev), torch.empty((B, S, H2, D), dtype=x.dtype, device=dev)
            ptr2, st2 = second.data_ptr(), _strides(second)
        d = _abi.Rotary.from_buffer_copy(_abi.ROTARY_FORMAT.pack(
            code, kind, inverse, pos.element_size(), B, S, D, 2 * turns, H, H2, *_strides(one), *st2,
            0 if len(at) == 1 else pos.stride(0), pos.stride(-1), scale, 0))
        _abi.check(_abi.lib().lego_rotary(C.byref(d), one.data_ptr(), ptr2, y1.data_ptr(), _ptr(y2), pos.data_ptr(),
                                          fr.data_ptr(), _stream_on(dev)), "lego_rotary")
        return [_like_input(y1, x)] if two is None else [_like_input(y1, x), _like_input(y2, two)]


def _first_order(backward):
    """A backward pass through which no gradient goes.  What says so costs 4 us a call (of 129 of a rotary
    training step of 64 tokens) and is only needed where a graph of the backward pass is made."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


class LEGORotary(torch.autograd.Function):
    """``LEGORotary.apply(q, k, positions, freqs, pairs, scale)``; ``k`` may be None."""

    @classmethod
    def apply(cls, q, k, positions, freqs, pairs, scale):
        _check_tangents(q, k, freqs)
        _check_constants(freqs=freqs, scale=scale)
        return super().apply(q, k, positions, freqs, pairs, scale)

    @staticmethod
    def forward(ctx, q, k, positions, freqs, pairs, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, freqs)
        ctx.pairs, ctx.scale = pairs, scale
        out = _rotary([q] if k is None else [q, k], positions, freqs, pairs, scale, False)
        return (out[0], out[1] if k is not None else None)

    @staticmethod
    @_first_order
    def backward(ctx, dq, dk):
        positions, freqs = ctx.saved_tensors
        given = [g for g in (dq, dk) if g is not None]
        back = iter(_rotary(given, positions, freqs, ctx.pairs, ctx.scale, True) if given else ())
        return tuple(None if g is None else next(back) for g in (dq, dk)) + (None,) * 4


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, freqs: torch.Tensor, *,
           pairs: str = "half", scale: float = 1.0):
    """Queries ``[B, S, Hq, D]`` and keys ``[B, S, Hk, D]`` turned by their positions, in one launch:
    pair ``p`` of the first ``2 len(freqs)`` values of every head by the angle ``position * freqs[p]``
    (``rotary_frequencies``), the rest copied.  ``pairs``: ``"half"`` pairs value p with value p + len(freqs),
    ``"interleaved"`` 2p with 2p + 1.  ``positions``: int32 or int64 ``[B, S]`` or ``[S]``.  ``scale``
    multiplies the turned values.  Differentiable in q and k (``freqs`` and ``scale`` are constants).  Returns ``(q, k)``, or q alone when
    ``k`` is None.  float16, bfloat16 or float32, any strides with a contiguous last axis."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = LEGORotary.apply(q, k, positions, freqs, pairs, scale)
        return out[0] if k is None else out
    _check_constants(freqs=freqs, scale=scale)
    out = _rotary([q] if k is None else [q, k], positions, freqs, pairs, scale, False)
    return out[0] if k is None else tuple(out)


def _attention_desc(q, k, v, causal, prefix, documents, softcap, slopes, scale):
    """Checks of an attention call; ``(device, descriptor, tensors it refers to)`` with q, k, v first."""
    _check_tangents(q, k, v, slopes)
    code = _ATTN_TYPES.get(q.dtype)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention takes q [B, Sq, Hq, D] and k, v [B, Sk, Hk, D]")
    if code is None or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("attention takes float16 or bfloat16 tensors of one type")
    B, Sq, Hq, D = q.shape
    Bk, Sk, Hk, Dk = k.shape
    if Bk != B or Dk != D or k.shape != v.shape:
        raise ValueError("q, k, v must agree in batch and head size, k and v in shape")
    if Hk < 1 or Hq % Hk:
        raise ValueError(f"{Hq} query heads cannot share {Hk} key heads evenly")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError("head size must be a multiple of 8 up to 128")
    if prefix is not None:
        if not causal:
            raise ValueError("a prefix needs causal=True")
        _check_int32(prefix, "prefix", (B,))
    if documents is not None:
        if Sq > Sk:
            raise ValueError("documents need as many keys as queries at least")
        _check_int32(documents, "documents", (B, Sk))
    if slopes is not None:
        _check_slopes(slopes, Hq)
    scale, softcap = _scores(scale, softcap, D)
    dev = _same_device(q, k, v, prefix, documents, slopes)
    (qd, q_st), (kd, k_st), (vd, v_st) = _strided(q, dev), _strided(k, dev), _strided(v, dev)
    keep = [qd, kd, vd]
    options = (0, 0, 0)
    if slopes is not None or prefix is not None or documents is not None:
        given = [_optional(t, dev) for t in (slopes, prefix, documents)]
        options = [t.data_ptr() if t is not None else 0 for t in given]
        keep += given
    d = _abi.Attention.from_buffer_copy(_abi.ATTENTION_FORMAT.pack(
        code, 1 if causal else 0, B, Sq, Sk, Hq, Hk, D, *q_st, *k_st, *v_st, scale, softcap, *options))
    return dev, d, keep


def _attention_workspace(d, backward, dev):
    n = _abi.lib().lego_attention_workspace_bytes(C.byref(d), backward)
    if n < 0:
        _abi.check(n, "lego_attention_workspace_bytes")
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None, n


def _attention_fwd(q, k, v, causal, prefix, documents, softcap, slopes, scale, low):
    """``(o, lse, what o's rounding left or None)``."""
    dev, d, keep = _attention_desc(q, k, v, causal, prefix, documents, softcap, slopes, scale)
    B, Sq, Hq, _ = shape = q.shape
    with _on(dev):
        o = torch.empty(shape, dtype=q.dtype, device=dev)
        lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=dev)
        o_low = torch.empty(shape, dtype=q.dtype, device=dev) if low else None
        if k.shape[1] == 0:
            o.zero_()
            lse.fill_(-math.inf)
            o_low = None
        elif o.numel():
            ws, n = _attention_workspace(d, 0, dev)
            _abi.check(_abi.lib().lego_attention_fwd(C.byref(d), keep[0].data_ptr(), keep[1].data_ptr(), keep[2].data_ptr(),
                                                     o.data_ptr(), _ptr(o_low), lse.data_ptr(), _ptr(ws), n, _stream_on(dev)),
                       "lego_attention_fwd")
        if q.is_cuda:
            return o, lse, o_low
        return _to_host(o), _to_host(lse), None if o_low is None else _to_host(o_low)


def attention_fwd(q, k, v, causal=False, prefix=None, documents=None, softcap=0.0, slopes=None, scale=None):
    """Attention forward: ``(o, lse)``, see ``attention``; lse is float32 ``[B, Hq, Sq]``."""
    _check_constants(slopes=slopes, softcap=softcap, scale=scale)
    return _attention_fwd(q, k, v, causal, prefix, documents, softcap, slopes, scale, False)[:2]


def attention_bwd(do, q, k, v, o, lse, causal=False, prefix=None, documents=None, softcap=0.0, slopes=None, scale=None,
                  o_low=None):
    """Attention backward from what ``attention_fwd`` took and gave: ``(dq, dk, dv)``, contiguous,
    the same bits on every run.  ``o_low``: what the rounding of o left, as ``LEGOAttention`` keeps it;
    without it the gradients of rows with one large weight carry that rounding too."""
    _check_tangents(do, o, lse, o_low)
    _check_constants(slopes=slopes, softcap=softcap, scale=scale)
    dev, d, keep = _attention_desc(q, k, v, causal, prefix, documents, softcap, slopes, scale)
    _same_device(do, o, lse, o_low, keep[0])
    B, Sq, Hq, _ = q.shape
    if do.shape != q.shape or o.shape != q.shape or tuple(lse.shape) != (B, Hq, Sq) or (
            o_low is not None and o_low.shape != q.shape):
        raise ValueError("do and o must have q's shape, lse [B, Hq, Sq]")
    if do.dtype != q.dtype or o.dtype != q.dtype or lse.dtype != torch.float32 or (
            o_low is not None and o_low.dtype != q.dtype):
        raise ValueError("do and o must have q's type, lse float32")
    with _on(dev):
        dod, od, lsed = _dense(do, dev), _dense(o, dev), _dense(lse, dev)
        lowd = None if o_low is None else _dense(o_low, dev)
        dq, dk, dv = (torch.empty(t.shape, dtype=q.dtype, device=dev) for t in (q, k, v))
        if dq.numel() == 0 or dk.numel() == 0:
            for g in (dq, dk, dv):
                g.zero_()
        else:
            ws, n = _attention_workspace(d, 1, dev)
            _abi.check(_abi.lib().lego_attention_bwd(C.byref(d), keep[0].data_ptr(), keep[1].data_ptr(), keep[2].data_ptr(),
                                                     od.data_ptr(), _ptr(lowd), lsed.data_ptr(), dod.data_ptr(), dq.data_ptr(),
                                                     dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), n, _stream_on(dev)),
                       "lego_attention_bwd")
        return _like_input(dq, q), _like_input(dk, k), _like_input(dv, v)


class LEGOAttention(torch.autograd.Function):
    """``LEGOAttention.apply(q, k, v, causal, prefix, documents, softcap, slopes, scale)`` -> ``(o, lse)``."""

    @classmethod
    def apply(cls, q, k, v, causal, prefix, documents, softcap, slopes, scale):
        _check_tangents(q, k, v, slopes)
        _check_constants(slopes=slopes, softcap=softcap, scale=scale)
        return super().apply(q, k, v, causal, prefix, documents, softcap, slopes, scale)

    @staticmethod
    def forward(ctx, q, k, v, causal, prefix, documents, softcap, slopes, scale):
        o, lse, o_low = _attention_fwd(q, k, v, causal, prefix, documents, softcap, slopes, scale, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(lse)
        ctx.save_for_backward(q, k, v, o, lse, o_low, prefix, documents, slopes)
        ctx.rest = (causal, softcap, scale)
        return o, lse

    @staticmethod
    @_first_order
    def backward(ctx, do, _):
        if do is None:
            return (None,) * 9
        q, k, v, o, lse, o_low, prefix, documents, slopes = ctx.saved_tensors
        causal, softcap, scale = ctx.rest
        return (*attention_bwd(do, q, k, v, o, lse, causal, prefix, documents, softcap, slopes, scale, o_low), *(None,) * 6)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False,
              prefix: Optional[torch.Tensor] = None, documents: Optional[torch.Tensor] = None, softcap: float = 0.0,
              slopes: Optional[torch.Tensor] = None, scale: Optional[float] = None, return_lse: bool = False):
    """``softmax(scores) v`` of q ``[B, Sq, Hq, D]`` over k, v ``[B, Sk, Hk, D]`` (Hq a multiple of Hk;
    float16 or bfloat16, D a multiple of 8 up to 128), without the scores ever in memory.

    Query i stands at position ``i + Sk - Sq`` of the keys.  Scores are ``scale q.k`` (default
    ``D ** -0.5``), bent by ``softcap * tanh(. / softcap)`` when ``softcap`` is positive, minus
    ``slopes[h] * |position - j|`` when ``slopes`` (float32 ``[Hq]``) is given.  ``causal``: a query sees the
    keys up to its position, and those before ``prefix[b]`` (int32 ``[B]``) too.  ``documents`` (int32
    ``[B, Sk]``): only keys of the query's own document; negative numbers mark padding, which sees and
    shows nothing and whose values are not used.  A query that sees no key gets zeros.

    Differentiable in q, k and v (``slopes``, ``softcap`` and ``scale`` are constants).  ``return_lse``: also the logarithm of each row's sum, float32
    ``[B, Hq, Sq]`` (no gradient).  Tokens that are not padding have to be finite, whoever sees them: a
    hidden one meets a weight of zero.  To capture a backward pass into a CUDA graph take
    ``torch.autograd.grad``, or keep no eager graph of the same leaves alive."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, lse = LEGOAttention.apply(q, k, v, causal, prefix, documents, softcap, slopes, scale)
    else:
        o, lse = attention_fwd(q, k, v, causal, prefix, documents, softcap, slopes, scale)
    return (o, lse) if return_lse else o


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                   lengths: torch.Tensor, parents: Optional[torch.Tensor] = None, *, softcap: float = 0.0,
                   slopes: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of drafted tokens q ``[B, T, Hq, D]`` (T up to 64) over a cache of pages
    ``[pages, page_size, Hk, D]``: the serving form of ``attention``, with the same scores.

    Place p of sequence b is slot ``p % page_size`` of page ``page_table[b, p // page_size]`` (int32).
    ``lengths`` (int32 ``[B]``) counts the tokens cached before the draft; the keys and values of
    drafted token t stand in place ``lengths[b] + t``.  A drafted token sees the cached tokens, the
    drafted ones it descends from and itself.  ``parents`` (int32 ``[B, T]``) names the draft token
    each one follows, -1 the cached text; None is a chain, so T = 1 is plain decoding.  A token whose
    parent is neither -1 nor an earlier token, or descends from such a one, is unused and gets zeros,
    as do all tokens of a sequence of negative length.  What the cache holds past a sequence's last
    place is not used.  No gradient."""
    _check_tangents(q, k_cache, v_cache, slopes)
    if q.dim() != 4 or k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("tree_attention takes q [B, T, Hq, D] and caches [pages, page_size, Hk, D]")
    code = _ATTN_TYPES.get(q.dtype)
    if code is None or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("tree_attention takes float16 or bfloat16 tensors of one type")
    B, T, Hq, D = q.shape
    pages, page_size, Hk, _ = k_cache.shape
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != D:
        raise ValueError("q and the caches must agree in head size, the caches in shape")
    if Hk < 1 or Hq % Hk:
        raise ValueError(f"{Hq} query heads cannot share {Hk} key heads evenly")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError("head size must be a multiple of 8 up to 128")
    if not 1 <= T <= _abi.MAX_DRAFT:
        raise ValueError(f"1 .. {_abi.MAX_DRAFT} drafted tokens per sequence")
    if page_table.dim() != 2 or pages < 1 or page_size < 1 or page_table.shape[1] < 1:
        raise ValueError("page_table must be int32 [B, pages of a sequence], the cache must not be empty")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise ValueError("tree_attention has no gradient: call it under torch.no_grad()")
    _check_constants(slopes=slopes, softcap=softcap, scale=scale)
    _check_int32(page_table, "page_table", (B, page_table.shape[1]))
    _check_int32(lengths, "lengths", (B,))
    if parents is not None:
        _check_int32(parents, "parents", (B, T))
    if slopes is not None:
        _check_slopes(slopes, Hq)
    scale, softcap = _scores(scale, softcap, D)
    dev = _same_device(q, k_cache, v_cache, page_table, lengths, parents, slopes)
    with _on(dev):
        table, lens = _ready(page_table, dev).contiguous(), _ready(lengths, dev).contiguous()
        par, sl = _optional(parents, dev), _optional(slopes, dev)
        (qd, q_st), (kd, k_st), (vd, v_st) = _strided(q, dev), _strided(k_cache, dev), _strided(v_cache, dev)
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if B == 0 or Hq == 0:
            return _like_input(o, q)
        n_table = table.shape[1]
        d = _abi.TreeAttention.from_buffer_copy(_abi.TREE_ATTENTION_FORMAT.pack(
            code, 0, B, T, Hq, Hk, D, pages, page_size, n_table, n_table, *q_st, *k_st, *v_st, scale, softcap))
        lib, ref = _abi.lib(), C.byref(d)
        n = lib.lego_tree_attention_workspace_bytes(ref)
        _abi.check(min(n, 0), "lego_tree_attention_workspace_bytes")
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _abi.check(lib.lego_tree_attention(ref, qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), table.data_ptr(),
                                           lens.data_ptr(), _ptr(par), _ptr(sl), o.data_ptr(), ws.data_ptr(), n,
                                           _stream_on(dev)), "lego_tree_attention")
        return _like_input(o, q)
