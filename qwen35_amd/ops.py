"""Thin torch-facing wrappers over the C ABI (device tensors in, device tensors out).

Every call goes straight to a HIP kernel of libqwen35_hip.so on the current
torch stream; nothing is computed on the host.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import QhipKvBatch, QhipKvCache, QhipLinear, QhipLinearBatch, QhipProfEntry, QhipRows, check, load

_GEOM = {8: (32, 34), 20: (32, 18), 12: (256, 144), 14: (256, 210), 13: (256, 176), 11: (256, 110),
         10: (256, 84), 23: (256, 136), 2: (32, 18), 3: (32, 20), 18: (256, 98), 21: (256, 110)}
# integers per 32-value block in the block-integer export: (sumi, sumy) for Q4_1
_NINTS_32 = {3: 2}
# integers per super-block in the block-integer export: (isum, summs) for
# Q4_K / Q5_K / Q2_K, one per 32-value block for IQ4_XS and the IQ3 formats, else one
_NINTS_SB = {12: 2, 13: 2, 10: 2, 23: 8, 18: 8, 21: 8}


def _stream(device: int | None = None) -> ctypes.c_void_p:
    """The current stream's handle on the current device (torch.cuda.current_stream builds a stream object first: 2.8 us)."""
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if device is None else device))


def _p(t: torch.Tensor) -> ctypes.c_void_p:
    assert t.is_cuda and t.is_contiguous()
    return ctypes.c_void_p(t.data_ptr())


def act_row_bytes(ttype: int, cols: int) -> int:
    n = load().qhip_act_row_bytes(ttype, cols)
    if n < 0:
        raise ValueError(f"bad (ttype={ttype}, cols={cols})")
    return n


def weight_row_bytes(ttype: int, cols: int) -> int:
    n = load().qhip_weight_row_bytes(ttype, cols)
    if n < 0:
        raise ValueError(f"bad (ttype={ttype}, cols={cols})")
    return n


def quantize_act(ttype: int, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [k, cols] f32 -> [k, act_row_bytes] uint8, the weight type's activation family."""
    x2 = x.reshape(-1, x.shape[-1])
    k, cols = x2.shape
    if out is None:
        out = torch.empty((k, act_row_bytes(ttype, cols)), dtype=torch.uint8, device=x.device)
    check("quantize_act", load().qhip_launch_quantize_act(ttype, _p(x2), _p(out), cols, k, _stream()))
    return out


def quantize_q8_0(x: torch.Tensor) -> torch.Tensor:
    n = x.numel()
    out = torch.empty(n // 32 * 34, dtype=torch.uint8, device=x.device)
    check("quantize_q8_0", load().qhip_launch_quantize_q8_0(_p(x), _p(out), n // 32, _stream()))
    return out


def quantize_q8_K(x: torch.Tensor) -> torch.Tensor:
    n = x.numel()
    out = torch.empty(n // 256 * 292, dtype=torch.uint8, device=x.device)
    check("quantize_q8_K", load().qhip_launch_quantize_q8_K(_p(x), _p(out), n // 256, _stream()))
    return out


def dequantize(ttype: int, w: torch.Tensor, nblocks: int) -> torch.Tensor:
    """f32 values of `nblocks` native blocks (bit-exact with the reference dequant)."""
    be = _GEOM[ttype][0]
    out = torch.empty(nblocks * be, dtype=torch.float32, device=w.device)
    check("dequantize", load().qhip_launch_dequantize(ttype, _p(w), _p(out), nblocks, _stream()))
    return out


def dequantize_row(ttype: int, wrow: torch.Tensor, cols: int) -> torch.Tensor:
    out = torch.empty(cols, dtype=torch.float32, device=wrow.device)
    check("dequantize_row", load().qhip_launch_dequantize_row(ttype, _p(wrow), _p(out), cols, _stream()))
    return out


def mul_mat(ttype: int, w: torch.Tensor, xq: torch.Tensor, rows: int, cols: int, tokens: int,
            path: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """out [tokens, rows] = W . xq_t (xq already quantized)."""
    if out is None:
        out = torch.empty((tokens, rows), dtype=torch.float32, device=w.device)
    check("mul_mat", load().qhip_launch_mul_mat(_p(w), _p(xq), _p(out), rows, cols, tokens, ttype,
                                                path, _stream()))
    return out


def mul_mat_work(rows: int, cols: int, tokens: int, ttype: int, device) -> torch.Tensor | None:
    """Zeroed split-K workspace for mul_mat_split / mul_mat_image (None when no split would be made)."""
    n = load().qhip_mul_mat_work_bytes(rows, cols, tokens, ttype)
    return torch.zeros(n, dtype=torch.uint8, device=device) if n > 0 else None


def mul_mat_split(ttype: int, w: torch.Tensor, xq: torch.Tensor, rows: int, cols: int, tokens: int,
                  work: torch.Tensor | None, path: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """mul_mat with a workspace: the MMQ of small grids splits K (deterministic slice order)."""
    if out is None:
        out = torch.empty((tokens, rows), dtype=torch.float32, device=w.device)
    check("mul_mat_work", load().qhip_launch_mul_mat_work(
        _p(w), _p(xq), _p(out), rows, cols, tokens, ttype, path, _p(work) if work is not None else None,
        work.numel() if work is not None else 0, _stream()))
    return out


def quantize_mul_mat_vec(ttype: int, w: torch.Tensor, x: torch.Tensor, rows: int, cols: int,
                         xq_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One launch: quantize f32 x (one token) inside the GEMV and multiply."""
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=w.device)
    check("quantize_mul_mat_vec", load().qhip_launch_quantize_mul_mat_vec(
        _p(w), _p(x), _p(xq_out) if xq_out is not None else None, _p(out), rows, cols, ttype, _stream()))
    return out


def quantize_mul_mat_vec_tuned(ttype: int, w: torch.Tensor, x: torch.Tensor, rows: int, cols: int,
                               lanes_per_row: int = 0, rows_per_lane: int = 0, workgroup_threads: int = 0,
                               xq_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The one-launch quantize + GEMV with an explicit shape (0 = pick)."""
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=w.device)
    check("quantize_mul_mat_vec_tuned", load().qhip_launch_quantize_mul_mat_vec_tuned(
        _p(w), _p(x), _p(xq_out) if xq_out is not None else None, _p(out), rows, cols, ttype, lanes_per_row,
        rows_per_lane, workgroup_threads, _stream()))
    return out


def split_work(rows: int, cols: int, device) -> torch.Tensor:
    """Zeroed workspace for quantize_mul_mat_vec_split (its counters must start at zero)."""
    n = load().qhip_quantize_mul_mat_vec_work_bytes(rows, cols)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def quantize_mul_mat_vec_split(ttype: int, w: torch.Tensor, x: torch.Tensor, rows: int, cols: int,
                               work: torch.Tensor, slice_values: int = 0, lanes_per_row: int = 0,
                               rows_per_lane: int = 0, xq_out: torch.Tensor | None = None,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """One launch, split over K: each workgroup quantizes and multiplies one slice of x."""
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=w.device)
    check("quantize_mul_mat_vec_split", load().qhip_launch_quantize_mul_mat_vec_split(
        _p(w), _p(x), _p(xq_out) if xq_out is not None else None, _p(out), rows, cols, ttype, slice_values,
        lanes_per_row, rows_per_lane, _p(work), work.numel(), _stream()))
    return out


def quantize_mul_mat_vec_split_noalloc(ttype: int, w: torch.Tensor, x: torch.Tensor, rows: int, cols: int,
                                       slice_values: int = 0, lanes_per_row: int = 0, rows_per_lane: int = 0,
                                       xq_out: torch.Tensor | None = None,
                                       out: torch.Tensor | None = None) -> torch.Tensor:
    """The split-K launch with the library's own per-device workspace (no allocation in the call)."""
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=w.device)
    check("quantize_mul_mat_vec_split_noalloc", load().qhip_launch_quantize_mul_mat_vec_split_noalloc(
        _p(w), _p(x), _p(xq_out) if xq_out is not None else None, _p(out), rows, cols, ttype, slice_values,
        lanes_per_row, rows_per_lane, _stream()))
    return out


def gemv_tuned(ttype: int, w: torch.Tensor, xq: torch.Tensor, rows: int, cols: int, tokens: int,
               lanes_per_row: int, tokens_per_pass: int, rows_per_lane: int = 1,
               out: torch.Tensor | None = None) -> torch.Tensor:
    if out is None:
        out = torch.empty((tokens, rows), dtype=torch.float32, device=w.device)
    check("gemv_tuned", load().qhip_launch_gemv_tuned(_p(w), _p(xq), _p(out), rows, cols, tokens,
                                                      ttype, lanes_per_row, tokens_per_pass,
                                                      rows_per_lane, _stream()))
    return out


def mmq_tuned(ttype: int, w: torch.Tensor, xq: torch.Tensor, rows: int, cols: int, tokens: int,
              tile_tokens: int = 0, tile_rows: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """The int8-MFMA tile path with an explicit workgroup tile (64 or 128 each, 0 = pick)."""
    if out is None:
        out = torch.empty((tokens, rows), dtype=torch.float32, device=w.device)
    check("mmq_tuned", load().qhip_launch_mmq_tuned(_p(w), _p(xq), _p(out), rows, cols, tokens, ttype,
                                                    tile_tokens, tile_rows, _stream()))
    return out


def mmq_image(ttype: int, w: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """The MMQ weight image of a Q4_K / Q6_K weight (sub-scales folded into two int8 planes)."""
    n = load().qhip_mmq_image_bytes(ttype, rows, cols)
    if n < 0:
        raise ValueError(f"no MMQ image for type {ttype} at cols={cols}")
    img = torch.empty(max(n, 16), dtype=torch.uint8, device=w.device)
    check("mmq_prepare", load().qhip_launch_mmq_prepare(ttype, _p(w), rows, cols, _p(img), _stream()))
    return img


def mul_mat_image(ttype: int, img: torch.Tensor, xq: torch.Tensor, rows: int, cols: int, tokens: int,
                  tile_tokens: int = 0, tile_rows: int = 0, work: torch.Tensor | None = None) -> torch.Tensor:
    out = torch.empty((tokens, rows), dtype=torch.float32, device=img.device)
    check("mul_mat_image", load().qhip_launch_mul_mat_image(
        _p(img), _p(xq), _p(out), rows, cols, tokens, ttype, tile_tokens, tile_rows,
        _p(work) if work is not None else None, work.numel() if work is not None else 0, _stream()))
    return out


def wd_image(ttype: int, w: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """The fragment image of a Q4_K / Q6_K / Q8_0 weight (the GGUF bytes permuted for the MMQ)."""
    n = load().qhip_wd_image_bytes(ttype, rows, cols)
    if n < 0:
        raise ValueError(f"no fragment image for type {ttype} at cols={cols}")
    img = torch.empty(max(n, 16), dtype=torch.uint8, device=w.device)
    check("wd_prepare", load().qhip_launch_wd_prepare(ttype, _p(w), rows, cols, _p(img), _stream()))
    return img


def mul_mat_wd_image(ttype: int, img: torch.Tensor, xq: torch.Tensor, rows: int, cols: int, tokens: int,
                     work: torch.Tensor | None = None) -> torch.Tensor:
    """out [tokens, rows] from the fragment image (Q6_K: 1..32 tokens; Q4_K, Q8_0: any)."""
    out = torch.empty((tokens, rows), dtype=torch.float32, device=img.device)
    check("mul_mat_wd_image", load().qhip_launch_mul_mat_wd_image(
        _p(img), _p(xq), _p(out), rows, cols, tokens, ttype,
        _p(work) if work is not None else None, work.numel() if work is not None else 0, _stream()))
    return out


def gemv_image(ttype: int, w: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """The GEMV weight image of an IQ4_NL / Q4_0 weight (same bytes per row, quant bytes 16-byte aligned)."""
    n = load().qhip_gemv_image_bytes(ttype, rows, cols)
    if n < 0:
        raise ValueError(f"no GEMV image for type {ttype} at cols={cols}")
    img = torch.empty(max(n, 16), dtype=torch.uint8, device=w.device)
    check("gemv_prepare", load().qhip_launch_gemv_prepare(ttype, _p(w), rows, cols, _p(img), _stream()))
    return img


def quantize_act_image(ttype: int, x: torch.Tensor) -> torch.Tensor:
    """f32 [tokens, cols] -> the split Q8_0 activation the GEMV image reads."""
    x = x.contiguous()
    cols = x.shape[-1]
    tokens = x.numel() // cols
    n = load().qhip_gemv_image_act_bytes(ttype, cols, tokens)
    if n < 0:
        raise ValueError(f"no split activation for type {ttype} at cols={cols}")
    out = torch.empty(max(n, 16), dtype=torch.uint8, device=x.device)
    check("quantize_act_image", load().qhip_launch_quantize_act_image(ttype, _p(x), _p(out), cols, tokens,
                                                                      _stream()))
    return out


def mul_mat_vec_image(ttype: int, img: torch.Tensor, xa: torch.Tensor, rows: int, cols: int,
                      rows_per_lane: int = 0) -> torch.Tensor:
    out = torch.empty(rows, dtype=torch.float32, device=img.device)
    check("mul_mat_vec_image", load().qhip_launch_mul_mat_vec_image(
        _p(img), _p(xa), _p(out), rows, cols, ttype, rows_per_lane, _stream()))
    return out


def block_ints(ttype: int, w: torch.Tensor, xq: torch.Tensor, rows: int, cols: int,
               tokens: int) -> torch.Tensor:
    be = _GEOM[ttype][0]
    nints = _NINTS_32.get(ttype, 1) * (cols // 32) if be == 32 else _NINTS_SB.get(ttype, 1) * (cols // 256)
    out = torch.empty((tokens, rows, nints), dtype=torch.int32, device=w.device)
    check("block_ints", load().qhip_launch_block_ints(_p(w), _p(xq), _p(out), rows, cols, tokens,
                                                      ttype, _stream()))
    return out


def ragged_offsets(lengths) -> tuple[list[int], int]:
    n = len(lengths)
    arr = (ctypes.c_int * n)(*lengths)
    off = (ctypes.c_int * (n + 1))()
    total = load().qhip_ragged_offsets(arr, n, off)
    if total < 0:
        raise ValueError("bad lengths")
    return list(off), total


def quantize_ragged(ttype: int, seqs: list[torch.Tensor], cols: int):
    """Pack + quantize several [L_i, cols] f32 sequences in one launch.
    Returns (xq_packed [total, act_row_bytes], offsets_dev [nseq+1] int32, total)."""
    lengths = [int(s.shape[0]) for s in seqs]
    off, total = ragged_offsets(lengths)
    dev = seqs[0].device
    ptrs = torch.tensor([s.data_ptr() for s in seqs], dtype=torch.int64, device=dev)
    off_d = torch.tensor(off, dtype=torch.int32, device=dev)
    xq = torch.empty((max(total, 1), act_row_bytes(ttype, cols)), dtype=torch.uint8, device=dev)
    check("quantize_ragged", load().qhip_launch_quantize_ragged(
        ttype, _p(ptrs), _p(off_d), len(seqs), total, cols, _p(xq), _stream()))
    return xq, off_d, total


def mul_mat_ragged(ttype: int, w: torch.Tensor, xq: torch.Tensor, off_d: torch.Tensor, nseq: int,
                   total: int, rows: int, cols: int) -> torch.Tensor:
    out = torch.empty((max(total, 1), rows), dtype=torch.float32, device=w.device)
    check("mul_mat_ragged", load().qhip_launch_mul_mat_ragged(
        _p(w), _p(xq), _p(out), rows, cols, _p(off_d), nseq, total, ttype, _stream()))
    return out[:total]


# ---- key/value cache in 8 bits ---------------------------------------------------------

_KV_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


# Launches go to the current device's stream, so a call's tensors have to lie on that device.
def _ints(name: str, t: torch.Tensor, device: int, dims: int = 1) -> int:
    if t.dtype != torch.int32 or t.dim() != dims or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor of {dims} dimension(s) on the current GPU")
    return t.data_ptr()


def _kv_rows(name: str, t: torch.Tensor, dim: int, device: int) -> int:
    """The GGUF type id of token rows [tokens, heads, dim] whose last dimension is contiguous."""
    if t.dim() != 3 or t.shape[2] != dim or t.stride(2) != 1 or t.get_device() != device or t.dtype not in _KV_TYPES:
        raise ValueError(f"{name}: a tensor [tokens, heads, {dim}] of f32, f16 or bf16 with contiguous heads on the current GPU")
    return _KV_TYPES[t.dtype]


def _c_ints(names: str, *numbers: int) -> None:
    """(ctypes would cut a number to its lowest 32 bits)"""
    for n in numbers:
        if not -0x80000000 <= n <= 0x7FFFFFFF:
            raise ValueError(f"{names}: {n} does not fit 32 bits")


def _kv_device(owner) -> int:
    """The current device, on which the tensors of the cache or step lie."""
    device = torch.cuda.current_device()
    if owner._device != device:
        raise ValueError(f"{type(owner).__name__}: on device {owner._device}, the current one is {device}")
    return device


class KvCache:
    """One layer's keys and values: int8 [blocks, kv_heads, block_size, head_dim] with f32 scales [blocks, kv_heads].
    Tensors of the same sizes may be put in their place (they are checked when they are set); the sizes are fixed."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        sizes = k.shape if k.dim() == 4 else (0, 0, 0, 0)
        self._c = QhipKvCache(None, None, None, None, sizes[0], sizes[2], sizes[1], sizes[3])
        self._ref = ctypes.byref(self._c)
        self.__dict__.update(zip(("num_blocks", "kv_heads", "block_size", "head_dim"), sizes), _device=k.get_device())
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    def __setattr__(self, name, value):
        if name in ("num_blocks", "kv_heads", "block_size", "head_dim"):
            raise AttributeError(f"{name}: fixed (another KvCache has other sizes)")
        if name in ("k", "v", "k_scale", "v_scale"):
            dtype, shape = torch.int8, (self.num_blocks, self.kv_heads, self.block_size, self.head_dim)
            if name in ("k_scale", "v_scale"):
                dtype, shape = torch.float32, shape[:2]
            if (not isinstance(value, torch.Tensor) or value.dtype != dtype or value.shape != shape or not value.is_cuda
                    or value.get_device() != self._device or not value.is_contiguous()):
                raise ValueError("k, v: contiguous int8 tensors [blocks, kv_heads, block_size, head_dim], k_scale, v_scale: "
                                 "f32 ones [blocks, kv_heads], all on one GPU")
            setattr(self._c, name, value.data_ptr())
        super().__setattr__(name, value)

    @classmethod
    def empty(cls, num_blocks: int, kv_heads: int, block_size: int, head_dim: int, device="cuda") -> "KvCache":
        shape = (num_blocks, kv_heads, block_size, head_dim)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))


class KvStep:
    """What kv_tables writes for a step of `nseq` sequences and `tokens` packed tokens: offsets [nseq + 1], kv_lens
    [nseq], slots and positions [tokens], taken [1].  Tensors put in their place are checked once, when they are set; the
    sizes are fixed."""

    def __init__(self, nseq: int, tokens: int, device="cuda"):
        self.__dict__.update(nseq=nseq, tokens=tokens)
        for name, n in self._entries().items():
            t = torch.empty(n, dtype=torch.int32, device=device)
            self.__dict__.setdefault("_device", t.get_device())
            setattr(self, name, t)

    def _entries(self) -> dict[str, int]:
        return {"offsets": self.nseq + 1, "kv_lens": self.nseq, "slots": self.tokens, "positions": self.tokens, "taken": 1}

    def __setattr__(self, name, value):
        if name in ("nseq", "tokens"):
            raise AttributeError(f"{name}: fixed (another KvStep has other sizes)")
        n = self._entries().get(name)
        if n is not None:
            if not isinstance(value, torch.Tensor) or value.shape != (n,):
                raise ValueError(f"{name}: {n} entries")
            if not value.is_cuda:
                raise ValueError(f"{name}: on a GPU")
            _ints(name, value, self._device)
        super().__setattr__(name, value)


def kv_tables(cached: torch.Tensor, new: torch.Tensor, free: torch.Tensor, table: torch.Tensor, block_size: int,
              step: KvStep, taken: torch.Tensor | None = None) -> KvStep:
    """Blocks and slots for `new` [nseq] tokens behind `cached` [nseq]: the new entries of `table` [nseq, width] come
    from `free`, from entry `taken` [1] on; `step` receives the rest.

    A sequence that falls back (rejected drafts) comes with a smaller `cached`; put its blocks behind that back into `free`
    (the entries before `taken` are spent) first, since their entries of `table` are overwritten."""
    nseq, dev = step.nseq, _kv_device(step)
    c, n, f, t = _ints("cached", cached, dev), _ints("new", new, dev), _ints("free", free, dev), _ints("table", table, dev, 2)
    rows, width = table.shape
    if cached.shape[0] != nseq or new.shape[0] != nseq or rows != nseq:
        raise ValueError(f"cached, new, table: {nseq} sequences")
    _c_ints("block_size", block_size)
    at = None if taken is None else _ints("taken", taken, dev)
    if taken is not None and taken.shape != (1,):
        raise ValueError("taken: one entry")
    check("kv_tables", load().qhip_launch_kv_tables(
        c, n, nseq, f, free.shape[0], at, block_size, t, width, step.tokens,
        step.offsets.data_ptr(), step.kv_lens.data_ptr(), step.slots.data_ptr(), step.positions.data_ptr(),
        step.taken.data_ptr(), _stream(dev)))
    return step


def kv_append(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Write k, v [tokens, kv_heads, head_dim] into `slots` [tokens] (-1: skip); the blocks' scales grow as needed."""
    dev = _kv_device(cache)
    tt = _kv_rows("k", k, cache.head_dim, dev)
    if _kv_rows("v", v, cache.head_dim, dev) != tt or k.shape != v.shape or k.shape[1] != cache.kv_heads or len(slots) != len(k):
        raise ValueError("k, v: one type, [tokens, kv_heads, head_dim]; slots: [tokens]")
    check("kv_append", load().qhip_launch_kv_append(
        cache._ref, tt, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
        _ints("slots", slots, dev), len(k), _stream(dev)))


def kv_read(cache: KvCache, blocks: torch.Tensor, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of whole blocks, [len(blocks), kv_heads, block_size, head_dim] each."""
    if dtype not in _KV_TYPES:
        raise ValueError("dtype: f32, f16 or bf16")
    dev = _kv_device(cache)
    ids = _ints("blocks", blocks, dev)
    shape = (len(blocks), cache.kv_heads, cache.block_size, cache.head_dim)
    k, v = torch.empty((2, *shape), dtype=dtype, device=blocks.device).unbind(0)
    check("kv_read", load().qhip_launch_kv_read(cache._ref, ids, len(blocks), _KV_TYPES[dtype], k.data_ptr(), v.data_ptr(),
                                                _stream(dev)))
    return k, v


def _kv_work(work: torch.Tensor, device: int) -> None:
    if work.dtype != torch.uint8 or work.dim() != 1 or work.get_device() != device or not work.is_contiguous():
        raise ValueError("work: a contiguous uint8 tensor on the current GPU (kv_attention_work)")


def kv_attention_work(cache: KvCache, q_heads: int, nseq: int, tokens: int, max_new: int, max_kv: int,
                      work: torch.Tensor | None = None) -> torch.Tensor | None:
    """Zeroed workspace for kv_attention of a batch of these sizes (None when nothing would be cut), or `work` itself, an
    earlier one, if it is large enough; with a smaller one, long sequences may go uncut."""
    _c_ints("nseq, tokens, max_new, max_kv", nseq, tokens, max_new, max_kv)
    b = QhipKvBatch(None, None, None, nseq, tokens, max_new, max_kv, 0)
    n = load().qhip_kv_attention_work_bytes(cache._ref, ctypes.byref(b), q_heads)
    if n < 0:
        raise ValueError(f"bad ({q_heads} query heads, {nseq} sequences, {tokens} tokens)")
    if work is not None:
        _kv_work(work, cache._device)
        if work.numel() >= n:
            return work
    return torch.zeros(n, dtype=torch.uint8, device=cache.k.device) if n > 0 else None


def kv_attention(q: torch.Tensor, cache: KvCache, table: torch.Tensor, offsets: torch.Tensor, kv_lens: torch.Tensor,
                 max_new: int, max_kv: int, scale: float | None = None, causal: bool = True, window: int = 0,
                 work: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of q [tokens, q_heads, head_dim] over the cached tokens of each row's sequence: (out, lse [tokens, q_heads]).

    Sequence i has rows offsets[i] .. offsets[i + 1] and kv_lens[i] cached tokens (its new ones included); no sequence
    has more than max_new rows or max_kv tokens.  scale: 1 / sqrt(head_dim) by default.  Rows at or past offsets[-1] are not
    written (where out or lse is not given: whatever the memory held).  work: kv_attention_work's tensor, whose first 32 KiB
    are zero before and after every call; calls that share one must not overlap (two streams need two).  f32 rows are good
    to f32; f16 and bf16 rows take softmax weights of 11 bits, which adds 2e-4 of an output to its own rounding."""
    dev = _kv_device(cache)
    tt, nseq = _kv_rows("q", q, cache.head_dim, dev), len(kv_lens)
    tokens, heads = q.shape[0], q.shape[1]
    if len(table) != nseq or len(offsets) != nseq + 1:
        raise ValueError(f"table: {nseq} rows, offsets: {nseq + 1}")
    if out is None:
        out = torch.empty((tokens, heads, cache.head_dim), dtype=q.dtype, device=q.device)
    elif _kv_rows("out", out, cache.head_dim, dev) != tt or out.shape != q.shape:
        raise ValueError("out: as q")
    if lse is None:
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device)
    elif lse.dtype != torch.float32 or lse.shape != (tokens, heads) or not lse.is_contiguous() or lse.get_device() != dev:
        raise ValueError("lse: f32 [tokens, q_heads]")
    if work is not None:
        _kv_work(work, dev)
    _c_ints("max_new, max_kv, window", max_new, max_kv, window)
    b = QhipKvBatch(_ints("offsets", offsets, dev), _ints("kv_lens", kv_lens, dev), _ints("table", table, dev, 2), nseq, tokens,
                    max_new, max_kv, table.shape[1])
    check("kv_attention", load().qhip_launch_kv_attention(
        cache._ref, ctypes.byref(b), tt, q.data_ptr(), q.stride(0), q.stride(1), heads,
        cache.head_dim ** -0.5 if scale is None else scale, int(causal), window, out.data_ptr(), out.stride(0), out.stride(1),
        lse.data_ptr(), None if work is None else work.data_ptr(), 0 if work is None else work.numel(), _stream(dev)))
    return out, lse


# ---- between a layer's products and its caches ------------------------------------------

# (each attribute of a tensor costs 0.1 to 0.3 us, and a call has up to twenty: shapes and strides are asked for once)
def _rows(name: str, t: torch.Tensor, device: int, shape: torch.Size, dtype: torch.dtype) -> QhipRows:
    """Rows of `shape` [tokens, dim] or [tokens, heads, dim] whose last dimension is contiguous."""
    stride = t.stride()
    if (t.dtype != dtype or t.shape != shape or t.get_device() != device or len(stride) not in (2, 3) or dtype not in _KV_TYPES
            or (stride[-1] != 1 and shape[-1] != 1) or (t.numel() > 0x7FFFFFFF and max(shape) > 0x7FFFFFFF)):
        raise ValueError(f"{name}: {list(shape)} of {dtype} (rows or heads of f32, f16 or bf16) with a contiguous last dimension on "
                         "the current GPU")
    return QhipRows(t.data_ptr(), stride[0], stride[1] if len(stride) == 3 else 0)


def _new_rows(shape: torch.Size, like: torch.Tensor) -> tuple[torch.Tensor, QhipRows]:
    t = torch.empty_like(like)  # (torch.empty with a type and a device takes three times as long)
    stride = t.stride()
    if t.shape != shape or stride[-1] != 1:  # (overlapping windows, for one, have an order of their own there)
        t = like.new_empty(shape)
        stride = t.stride()
    return t, QhipRows(t.data_ptr(), stride[0], stride[1] if len(stride) == 3 else 0)


def _rms_norm(x, weight, eps, residual, gate, out, ttype, xq):
    dev, shape, dtype = torch.cuda.current_device(), x.shape, x.dtype
    rows = _rows("x", x, dev, shape, dtype)
    if ttype is None and out is None:
        out, o = _new_rows(shape, x)
    else:
        o = None if out is None else _rows("out", out, dev, shape, dtype)
    r = None if residual is None else _rows("residual", residual, dev, shape, dtype)
    g = None if gate is None else _rows("gate", gate, dev, shape, dtype)
    heads, dim, w = shape[1] if len(shape) == 3 else 1, shape[-1], None
    if weight is not None:
        if weight.dtype != torch.float32 or weight.shape != (dim,) or weight.get_device() != dev or not weight.is_contiguous():
            raise ValueError(f"weight: a contiguous f32 tensor [{dim}] on the current GPU")
        w = weight.data_ptr()
    if ttype is not None:
        n = act_row_bytes(ttype, heads * dim)
        if xq is None:
            xq = torch.empty((shape[0], n), dtype=torch.uint8, device=x.device)
        elif xq.dtype != torch.uint8 or xq.shape != (shape[0], n) or not xq.is_contiguous() or xq.get_device() != dev:
            raise ValueError(f"xq: a contiguous uint8 tensor [{shape[0]}, {n}] on the current GPU")
    check("rms_norm", load().qhip_launch_rms_norm(
        _KV_TYPES[dtype], rows, r, g, w, eps, o, ttype or 0, None if xq is None else xq.data_ptr(), shape[0], heads, dim,
        _stream(dev)))
    return out if ttype is None else xq


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float, residual: torch.Tensor | None = None,
             gate: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension of x [tokens, dim] or [tokens, heads, dim].

    residual: x is added to it in place, and the sum is normalised.  gate: the result is multiplied by gate / (1 +
    exp(-gate)).  weight: f32 [dim].  out may be x or gate."""
    return _rms_norm(x, weight, eps, residual, gate, out, None, None)


def rms_norm_quantize(ttype: int, x: torch.Tensor, weight: torch.Tensor | None, eps: float, residual: torch.Tensor | None = None,
                      gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      xq: torch.Tensor | None = None) -> torch.Tensor:
    """rms_norm with its f32 result as the activation rows of weight type `ttype` (uint8 [tokens, act_row_bytes], the bytes
    that quantize_act makes of it); out: the unquantized result as well."""
    return _rms_norm(x, weight, eps, residual, gate, out, ttype, xq)


class RopeTable:
    """The frequencies of rotary positions: pair i of the first `rot_dim` values of a head turns by position * base^(-2 i /
    rot_dim), scaled for contexts `factor` times the trained one: "linear", "ntk" or "yarn" (which blends between the pairs
    that turn `fast` and `slow` times over `original` positions).  steps: an int64 tensor [rot_dim / 2], which another may
    replace (rope checks it and takes its address at each call); rot_dim is fixed."""

    SCALINGS = {None: 0, "linear": 1, "ntk": 2, "yarn": 3}

    def __init__(self, rot_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0, original: int = 0,
                 fast: float = 32.0, slow: float = 1.0, device="cuda"):
        if scaling not in self.SCALINGS:
            raise ValueError(f"scaling: one of {list(self.SCALINGS)}")
        _c_ints("rot_dim, original", rot_dim, original)
        steps, gain = (ctypes.c_ulonglong * max(rot_dim // 2, 1))(), ctypes.c_float()
        check("rope_steps", load().qhip_rope_steps(rot_dim, base, self.SCALINGS[scaling], factor, original, fast, slow, steps,
                                                   ctypes.byref(gain)))
        self.__dict__.update(rot_dim=rot_dim)
        self.gain = gain.value
        self.steps = torch.frombuffer(steps, dtype=torch.int64).to(device)

    def __setattr__(self, name, value):
        if name == "rot_dim":
            raise AttributeError("rot_dim: fixed (another RopeTable has another)")
        super().__setattr__(name, value)

    @property
    def device(self) -> int:
        return self.steps.get_device()


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: RopeTable, interleaved: bool = False,
         q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q [tokens, q_heads, dim] and k [tokens, k_heads, dim] (or None) with the first table.rot_dim values of every head
    turned by their token's position (int32 [tokens], KvStep.positions).

    Pairs are values i and i + rot_dim / 2, interleaved: 2 i and 2 i + 1.  q_out may be q, and k_out k."""
    dev, shape, dtype = torch.cuda.current_device(), q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError("q: [tokens, q_heads, dim]")
    tokens, q_heads, dim = shape
    qr, kr, ko, k_heads = _rows("q", q, dev, shape, dtype), None, None, 0
    if q_out is None:
        q_out, qo = _new_rows(shape, q)
    else:
        qo = _rows("q_out", q_out, dev, shape, dtype)
    if k is not None:
        k_shape = k.shape
        if len(k_shape) != 3 or k_shape[0] != tokens or k_shape[2] != dim:
            raise ValueError(f"k: [{tokens}, k_heads, {dim}]")
        k_heads, kr = k_shape[1], _rows("k", k, dev, k_shape, dtype)
        if k_out is None:
            k_out, ko = _new_rows(k_shape, k)
        else:
            ko = _rows("k_out", k_out, dev, k_shape, dtype)
    if positions.shape != (tokens,):
        raise ValueError(f"positions: {tokens} entries")
    steps, rot_dim = table.steps, table.rot_dim
    if steps.dtype != torch.int64 or steps.shape != (rot_dim // 2,) or steps.get_device() != dev or not steps.is_contiguous():
        raise ValueError(f"table: steps, a contiguous int64 tensor [{rot_dim // 2}] on the current GPU")
    check("rope", load().qhip_launch_rope(
        _KV_TYPES[dtype], qr, qo, q_heads, kr, ko, k_heads, dim, rot_dim, steps.data_ptr(), table.gain, int(interleaved),
        _ints("positions", positions, dev), tokens, _stream(dev)))
    return q_out, k_out


def _linear_states(states: torch.Tensor, device: int) -> torch.Size:
    shape = states.shape
    if states.dtype != torch.float32 or len(shape) != 4 or states.get_device() != device or not states.is_contiguous():
        raise ValueError("states: a contiguous f32 tensor [states, v_heads, key_dim, value_dim] on the current GPU")
    return shape


def _linear_work(work: torch.Tensor, device: int) -> int:
    if work.dtype != torch.uint8 or work.dim() != 1 or work.get_device() != device or not work.is_contiguous() or not work.numel():
        raise ValueError("work: a contiguous uint8 tensor on the current GPU, not empty (linear_attention_work)")
    return work.numel()


def linear_attention_work(states: torch.Tensor, q: torch.Tensor, nseq: int, max_new: int, delta: bool = True,
                          work: torch.Tensor | None = None) -> torch.Tensor | None:
    """Workspace for linear_attention of q's tokens, or `work` itself, an earlier one, if it is large enough; None where the
    call needs none (few new tokens a sequence).  What it holds is of no use behind the call, and it need not be cleared;
    calls that may run at once, captured ones too, each take their own."""
    dev = torch.cuda.current_device()
    shape = _linear_states(states, dev)
    tt = _kv_rows("q", q, shape[2], dev)
    _c_ints("nseq, max_new", nseq, max_new)
    b = QhipLinearBatch(None, None, None, nseq, q.shape[0], max_new, shape[0], q.shape[1], *shape[1:])
    n = load().qhip_linear_attention_work_bytes(b, tt, int(delta))
    if n < 0:
        raise ValueError(f"bad (states {list(shape)}, q {list(q.shape)}, {nseq} sequences)")
    if work is not None and _linear_work(work, dev) >= n:
        return work
    return torch.empty(n, dtype=torch.uint8, device=states.device) if n > 0 else None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, states: torch.Tensor,
                     slots: torch.Tensor, offsets: torch.Tensor, max_new: int, beta: torch.Tensor | None = None,
                     source: torch.Tensor | None = None, scale: float | None = None, work: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Linear attention of packed tokens over states [n, v_heads, key_dim, value_dim] (f32): with a = exp(log_decay),
    S <- a S + k^T u and out = scale q S, where u = v, or with `beta` (the delta rule) beta (v - k a S).

    q, k [tokens, k_heads, key_dim], v [tokens, v_heads, value_dim]; log_decay, beta: f32 [tokens, v_heads].  Sequence i has
    tokens offsets[i] .. offsets[i + 1], at most max_new, starts from state source[i] (-1: zeros; by default slots[i]) and
    leaves its last state in slots[i] (-1: nowhere); no state that a sequence writes may be another's in the same call.
    scale: 1 / sqrt(key_dim) by default.  Sums are f32 or more whatever the rows' type, and an output is rounded once, to it.
    Rows at or past offsets[-1] are not written.
    work: linear_attention_work's; with it sequences of more than a few tokens go in chunks of 64, several times as fast,
    without it (None) token by token."""
    dev, q_shape, dtype = torch.cuda.current_device(), q.shape, q.dtype
    n, v_heads, dk, dv = _linear_states(states, dev)
    if len(q_shape) != 3 or q_shape[2] != dk:
        raise ValueError(f"q: [tokens, k_heads, {dk}]")
    tokens, k_heads, _ = q_shape
    v_shape = torch.Size((tokens, v_heads, dv))
    qr, kr, vr = _rows("q", q, dev, q_shape, dtype), _rows("k", k, dev, q_shape, dtype), _rows("v", v, dev, v_shape, dtype)
    if out is None:
        out, o = _new_rows(v_shape, v)
    else:
        o = _rows("out", out, dev, v_shape, dtype)
    numbers = []
    for name, t in (("log_decay", log_decay), ("beta", beta)):
        if t is None:
            numbers += [None, 0]
            continue
        stride = t.stride()
        if t.dtype != torch.float32 or t.shape != v_shape[:2] or t.get_device() != dev or (stride[1] != 1 and v_heads > 1):
            raise ValueError(f"{name}: f32 [{tokens}, {v_heads}] with a contiguous last dimension on the current GPU")
        numbers += [t.data_ptr(), stride[0]]
    nseq = slots.shape[0] if slots.dim() == 1 else -1
    if offsets.shape != (nseq + 1,) or (source is not None and source.shape != (nseq,)):
        raise ValueError("slots [n], offsets [n + 1], source [n]")
    _c_ints("max_new", max_new)
    b = QhipLinearBatch(_ints("offsets", offsets, dev), _ints("slots", slots, dev), None if source is None else _ints("source", source, dev),
                        nseq, tokens, max_new, n, k_heads, v_heads, dk, dv)
    at, size = (None, 0) if work is None else (work.data_ptr(), _linear_work(work, dev))
    check("linear_attention", load().qhip_launch_linear_attention(
        b, _KV_TYPES[dtype], qr, kr, vr, *numbers, dk ** -0.5 if scale is None else scale, states.data_ptr(), o, at, size,
        _stream(dev)))
    return out


class Backend:
    """Python handle on the C++ backend (the Exec-slot mirror)."""

    def __init__(self, device: int = 0):
        lib = load()
        err = ctypes.c_int(0)
        self._h = lib.qhip_backend_create(device, ctypes.byref(err))
        if not self._h:
            check("backend_create", err.value or -1)
        self.lib = lib
        check("set_stream", lib.qhip_backend_set_stream(self._h, _stream()))

    def close(self):
        if self._h:
            self.lib.qhip_backend_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def name(self) -> str:
        return self.lib.qhip_backend_name(self._h).decode()

    def load_linear(self, ttype: int, rows: int, cols: int, host_bytes) -> QhipLinear:
        import numpy as np
        buf = np.ascontiguousarray(host_bytes, dtype=np.uint8)
        lin = QhipLinear()
        check("load_linear", self.lib.qhip_backend_load_linear(
            self._h, ttype, rows, cols, ctypes.c_void_p(buf.ctypes.data), ctypes.byref(lin)))
        return lin

    def wrap_linear(self, ttype: int, rows: int, cols: int, dev: torch.Tensor) -> QhipLinear:
        lin = QhipLinear()
        check("wrap_linear", self.lib.qhip_backend_wrap_linear(self._h, ttype, rows, cols, _p(dev),
                                                               ctypes.byref(lin)))
        return lin

    def free_linear(self, w: QhipLinear) -> None:
        self.lib.qhip_backend_free_linear(self._h, ctypes.byref(w))

    def prepare_linear(self, w: QhipLinear) -> int:
        """Build the weight's GEMV / MMQ image now: 0 built / nothing to build, -1 not built."""
        rc = self.lib.qhip_backend_prepare_linear(self._h, ctypes.byref(w))
        if rc not in (0, -1):
            check("prepare_linear", rc)
        return rc

    def set_mmq_images(self, on: bool) -> None:
        check("set_mmq_images", self.lib.qhip_backend_set_mmq_images(self._h, int(bool(on))))

    def set_gemv_images(self, on: bool) -> None:
        check("set_gemv_images", self.lib.qhip_backend_set_gemv_images(self._h, int(bool(on))))

    def set_mem_budget(self, nbytes: int) -> None:
        check("set_mem_budget", self.lib.qhip_backend_set_mem_budget(self._h, nbytes))

    def mem_placed(self) -> int:
        return int(self.lib.qhip_backend_mem_placed(self._h))

    def matvec(self, out: torch.Tensor, w: QhipLinear, x: torch.Tensor) -> None:
        check("matvec", self.lib.qhip_backend_matvec(self._h, _p(out), ctypes.byref(w), _p(x)))

    def matvec_pair(self, out: torch.Tensor, a: QhipLinear, b: QhipLinear, x: torch.Tensor) -> None:
        check("matvec_pair", self.lib.qhip_backend_matvec_pair(self._h, _p(out), ctypes.byref(a),
                                                               ctypes.byref(b), _p(x)))

    def matvec_batch_k(self, out: torch.Tensor, w: QhipLinear, xk: torch.Tensor, k: int) -> None:
        check("matvec_batch_k", self.lib.qhip_backend_matvec_batch_k(self._h, _p(out),
                                                                     ctypes.byref(w), _p(xk), k))

    def dequant_row(self, out: torch.Tensor, w: QhipLinear, row: int) -> None:
        check("dequant_row", self.lib.qhip_backend_dequant_row(self._h, _p(out), ctypes.byref(w), row))

    def sync(self) -> None:
        check("sync", self.lib.qhip_backend_sync(self._h))

    def set_stream(self, stream) -> None:
        """Launch on `stream` (a torch stream or a raw handle) from now on."""
        h = getattr(stream, "cuda_stream", stream)
        check("set_stream", self.lib.qhip_backend_set_stream(self._h, ctypes.c_void_p(h)))

    def set_act_memo(self, on: bool) -> None:
        check("set_act_memo", self.lib.qhip_backend_set_act_memo(self._h, int(bool(on))))

    def act_invalidate(self) -> None:
        self.lib.qhip_backend_act_invalidate(self._h)

    def act_stats(self) -> tuple[int, int]:
        hits, misses = ctypes.c_ulonglong(0), ctypes.c_ulonglong(0)
        check("act_stats", self.lib.qhip_backend_act_stats(self._h, ctypes.byref(hits),
                                                           ctypes.byref(misses)))
        return hits.value, misses.value

    def step_begin(self, pos: int) -> None:
        self.lib.qhip_backend_step_begin(self._h, pos)

    def step_end(self) -> None:
        self.lib.qhip_backend_step_end(self._h)

    def describe(self) -> str:
        return self.lib.qhip_backend_describe(self._h).decode()

    def set_profiling(self, on: bool) -> None:
        check("set_profiling", self.lib.qhip_backend_set_profiling(self._h, int(bool(on))))

    def prof_entries(self) -> list[dict]:
        """The device-time table, largest total first (waits for outstanding timings)."""
        n = self.lib.qhip_backend_prof_entries(self._h, None, 0)
        check("prof_entries", 0 if n >= 0 else n)
        arr = (QhipProfEntry * max(n, 1))()
        m = self.lib.qhip_backend_prof_entries(self._h, arr, n)
        assert m == n
        return [{f: getattr(arr[i], f) for f, _ in QhipProfEntry._fields_} for i in range(n)]

    def prof_report(self) -> str:
        n = self.lib.qhip_backend_prof_report(self._h, None, 0)
        assert n >= 0
        buf = ctypes.create_string_buffer(n + 1)
        assert self.lib.qhip_backend_prof_report(self._h, buf, n + 1) == n
        return buf.value.decode()

    def prof_untimed(self) -> int:
        return int(self.lib.qhip_backend_prof_untimed(self._h))

    def prof_reset(self) -> None:
        self.lib.qhip_backend_prof_reset(self._h)
