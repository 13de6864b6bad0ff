"""pagedkv -- Python front end of libpagedkv, the MI355X paged-KV engine.

Mirrors the reference's host API of the candle `engine = "paged"` path
(crates/ai-engine-candle/src/paged/{block_table,attention}.rs) on top of the
C ABI in include/pagedkv.h:

  BlockAllocator / BlockTable   block_table.rs:5-58 (C++ host code)
  PagedKvCache                  the reference's Vec<KvPool> (engine.rs:70-72)
  PagedKvCache.layer(l) -> KvPool  KvPool::{write, gather_seq} (attention.rs:39-97)
  KvPool.decode_attention       build_mask + sdpa of the decode step
                                (attention.rs:11-28,100-136, transformer.rs:271-292)
  KvPool.prefill_attention      prefill_seq's attention (transformer.rs:139-196)

torch tensors are used only as device memory and for the current stream.
"""
from __future__ import annotations

import collections
import contextlib
import ctypes
import sys
import math
from typing import Sequence

from ._lib import (BF16, F16, F32, K, V, CapacityError, PagedKvError, check, lib,
                   LIB_PATH)

__all__ = [
    "BlockAllocator", "BlockTable", "PagedKvCache", "KvPool", "Rope", "rope_tables_host",
    "CapacityError",
    "PagedKvError", "F32", "F16", "BF16", "lib", "LIB_PATH", "torch_dtype",
    "pkv_dtype", "StepTables", "step_tables", "verify_drafts",
]


# ---------------------------------------------------------------------------
# host block bookkeeping (C++), block_table.rs:5-58
# ---------------------------------------------------------------------------
class BlockTable:
    """One sequence's ordered physical block ids (block_table.rs:10-14)."""

    def __init__(self) -> None:
        self._h = lib().pkv_table_new()
        if not self._h:
            raise MemoryError("pkv_table_new")

    def __del__(self, _finalizing=sys.is_finalizing) -> None:
        h = getattr(self, "_h", None)
        if h and not _finalizing():
            lib().pkv_table_free(h)
            self._h = None

    @property
    def blocks(self) -> list[int]:
        n = lib().pkv_table_len(self._h)
        if n == 0:
            return []
        ptr = lib().pkv_table_blocks(self._h)
        return [ptr[i] for i in range(n)]

    def __len__(self) -> int:
        return int(lib().pkv_table_len(self._h))


class BlockAllocator:
    """Fixed-size block pool with a LIFO free list (block_table.rs:16-58)."""

    def __init__(self, num_blocks: int, block_size: int) -> None:
        self._h = lib().pkv_allocator_new(num_blocks, block_size)
        if not self._h:
            raise ValueError("pkv_allocator_new: bad arguments or out of memory")
        self.block_size = block_size

    def __del__(self, _finalizing=sys.is_finalizing) -> None:
        h = getattr(self, "_h", None)
        if h and not _finalizing():
            lib().pkv_allocator_free(h)
            self._h = None

    def free_count(self) -> int:
        return int(lib().pkv_allocator_free_count(self._h))

    def blocks_for(self, n_tokens: int) -> int:
        return int(lib().pkv_allocator_blocks_for(self._h, n_tokens))

    def ensure_capacity(self, table: BlockTable, n_tokens: int) -> None:
        """Raises CapacityError (nothing allocated) when the pool is short."""
        check(lib().pkv_allocator_ensure_capacity(self._h, table._h, n_tokens))

    def release(self, table: BlockTable) -> None:
        lib().pkv_allocator_release(self._h, table._h)

    def locate(self, table: BlockTable, pos: int) -> tuple[int, int]:
        blk = ctypes.c_uint32()
        slot = ctypes.c_size_t()
        rc = lib().pkv_allocator_locate(self._h, table._h, pos, ctypes.byref(blk),
                                        ctypes.byref(slot))
        if rc != 0:
            raise IndexError(f"position {pos} beyond the block table")
        return int(blk.value), int(slot.value)

    def slot(self, table: BlockTable, pos: int) -> int:
        b, s = self.locate(table, pos)
        return b * self.block_size + s


# ---------------------------------------------------------------------------
# device pool
# ---------------------------------------------------------------------------
def pkv_dtype(t) -> int:
    import torch
    m = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
    if t not in m:
        raise TypeError(f"unsupported dtype {t}")
    return m[t]


def torch_dtype(d: int):
    import torch
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[d]


def _stream_ptr(stream) -> int | None:
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    return int(stream.cuda_stream) or None


def _dev_ptr(t) -> int:
    return int(t.data_ptr())


def _i32(x, device):
    import torch
    if isinstance(x, torch.Tensor):
        t = x.to(device=device, dtype=torch.int32)
    else:
        t = torch.as_tensor(x, dtype=torch.int32).to(device)
    return t.contiguous()


def rope_tables_host(rope_dim: int, freq_base: float, max_seq: int):
    """Rope::new's cos/sin tables (rope.rs:14-23) computed by the library on
    the host: two float32 arrays (max_seq, rope_dim // 2)."""
    import numpy as np
    c = np.zeros((max_seq, rope_dim // 2), np.float32)
    s = np.zeros_like(c)
    check(lib().pkv_rope_tables_host(rope_dim, freq_base, max_seq, c.ctypes.data,
                                     s.ctypes.data), None)
    return c, s


def sample_draw(seed: int = 42) -> float:
    """StdRng::seed_from_u64(seed).gen::<f32>() (sample.rs:41-42), the fixed
    draw that sample() compares the cumulative probabilities with."""
    return float(lib().pkv_sample_draw(seed))


def sample(logits, temperatures=None, top_k: int | None = None, top_p: float | None = None,
           seed: int = 42, out=None, stream=None, exact: bool = True, routes=None):
    """Token per logits row on the device: argmax / sample() of sample.rs:12-55.
    logits: (batch, vocab) f32/f16/bf16 with unit stride along vocab;
    temperatures: (batch,) float32 on the device (None: all greedy).
    exact=True (pkv_sample_exact, the default since the engine needs the
    reference's tokens): the reference's f32 arithmetic bit for bit, so the
    token is the reference's on every row.  It takes its scratch on the
    stream for each call (freed in stream order after the launch; the library
    keeps up to 512 MiB of it per device until sample_trim()): 1 MiB per row for 16-bit logits (the row's runs of equal
    values); for f32 logits 8 bytes per logit (1 MiB per 128k-entry row),
    rows taken in rounds of at most 512 MiB.  top_p=None is the reference's
    None (no cut; passed as NaN), which differs from Some(1.0): with f32
    sums, 1.0 cuts where the running sum first reaches 1.0.
    exact=False (pkv_sample): faster, allocates only for rows split over
    several workgroups; sums the probabilities exactly, so a row can differ
    where the reference's f32 running sum lands within its rounding of r or
    top_p (top_p=None is 1.0 there, the same as no cut in exact sums).
    routes (exact=True only): a (batch,) int32 device tensor that receives
    the kernel that selected each row (pkv_sample_exact_routes: 0 argmax,
    1 buckets of f32 logits, 2 runs of equal 16-bit values, 3 radix sort).
    Returns (batch,) int32 on the device."""
    import torch
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be (batch, vocab) with unit stride along vocab")
    B, V = logits.shape
    dev = logits.device
    # The kernels run on `stream`: it first waits for the work queued so far
    # on the current stream (which produced the logits), and the temporaries
    # made here are allocated on it, so they are neither read early nor
    # reused before the launch has run.
    cur = torch.cuda.current_stream(dev)
    s = cur if stream is None else stream
    if s != cur:
        s.wait_stream(cur)
    if routes is not None and not exact:
        raise ValueError("routes are reported by the exact path only")
    if exact:  # top_p None is NaN; any other value is Some(top_p)
        fn, tp = lib().pkv_sample_exact, float("nan") if top_p is None else float(top_p)
    else:      # top_p None is 1.0 (no cut in exact arithmetic)
        fn, tp = lib().pkv_sample, 1.0 if top_p is None else float(top_p)
    extra = ()
    if routes is not None:
        if routes.dtype != torch.int32 or routes.numel() != B or not routes.is_contiguous():
            raise ValueError("routes must be a contiguous int32 tensor of one entry per row")
        fn, extra = lib().pkv_sample_exact_routes, (_dev_ptr(routes),)
    with torch.cuda.stream(s):
        if out is None:
            out = torch.empty(B, dtype=torch.int32, device=dev)
        t = None
        if temperatures is not None:
            t = torch.as_tensor(temperatures, dtype=torch.float32).to(dev).contiguous()
            if t.numel() != B:
                raise ValueError("temperatures must have one value per row")
        check(fn(_dev_ptr(logits) if V else None, pkv_dtype(logits.dtype),
                 logits.stride(0) if B > 1 else V, B, V,
                 _dev_ptr(t) if t is not None else None, top_k or 0, tp, seed, _dev_ptr(out),
                 *extra, _stream_ptr(s)), None)
    return out


def sample_trim() -> None:
    """Gives back the scratch that sample() keeps on the current device (at
    most 512 MiB; pkv_sample_trim)."""
    check(lib().pkv_sample_trim(), None)


def sample_expf(x):
    """expf as the exact sampler computes it (glibc's algorithm) for a float32
    device tensor; returns a new tensor."""
    import torch
    x = x.contiguous()
    if x.dtype != torch.float32:
        raise ValueError("float32 input expected")
    out = torch.empty_like(x)
    check(lib().pkv_sample_expf(_dev_ptr(x), _dev_ptr(out), x.numel(),
                                _stream_ptr(torch.cuda.current_stream(x.device))), None)
    return out


def _device_tensor(t, name: str, device, dtype, shape=None):
    """t, after a check that a kernel may read it as this."""
    if getattr(t, "device", None) != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    return t.contiguous()


def _i32_on(x, device):
    """_i32, at once for what is one already."""
    import torch
    if isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.device == device:
        return x.contiguous()
    return _i32(x, device)


_HERE = contextlib.nullcontext()


def _run_on(stream, device, tensors):
    """(raw stream to launch on, context in which to allocate and launch).
    Another stream than the current one first waits for the work queued on the
    current one, and the tensors' memory is not reused before it has run."""
    import torch
    if stream is None and torch.cuda.current_device() == device.index:
        # the handle alone: a Stream object costs 2 us of a 10 us call
        return torch._C._cuda_getCurrentRawStream(device.index) or None, _HERE
    cur = torch.cuda.current_stream(device)
    if stream is None or stream == cur:
        return _stream_ptr(cur), torch.cuda.device(device)
    if stream.device != device:
        raise ValueError(f"stream must be on {device}")
    stream.wait_stream(cur)
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return _stream_ptr(stream), torch.cuda.stream(stream)


def _workspace(nbytes: int, device):
    """Scratch of one call, from torch's allocator: it belongs to the call's
    stream, and to the graph's memory while that stream is captured."""
    import torch
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


StepTables = collections.namedtuple(
    "StepTables", "block_tables n_blocks free_count context_lens cu_q_lens positions "
                  "slot_mapping status")


def step_tables(seq_lens, new_lens, block_tables, n_blocks, free_list, free_count,
                block_size: int, num_blocks: int, max_tokens: int, stream=None) -> StepTables:
    """Block tables, slots and positions of a step from request lengths on the
    device (pkv_step_tables): request i, with seq_lens[i] tokens in n_blocks[i]
    blocks, writes new_lens[i] more; blocks that it lacks come from the end of
    free_list[: free_count] in request order (BlockAllocator.ensure_capacity).
    seq_lens, new_lens, n_blocks: (n,) int32, block_tables: (n, width) int32,
    free_list: (any,) int32, free_count: (1,) int32, all on one device;
    max_tokens: length of the step's token arrays (a host bound of the new
    tokens).  Nothing synchronises.  Returns new tensors:
      block_tables, n_blocks, free_count  for the next step
      context_lens (n,), cu_q_lens (n + 1,)
      positions, slot_mapping (max_tokens,), -1 past the step's tokens
      status (1,): 0, the number of blocks that the free list is short of, or
        -1 for lengths out of range; unless 0 the step is empty and tables,
        n_blocks and free_count are unchanged."""
    import torch
    if not isinstance(block_tables, torch.Tensor) or not block_tables.is_cuda:
        raise ValueError("block_tables must be a device tensor")
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be (n, width)")
    dev, i32 = block_tables.device, torch.int32
    n, width = block_tables.shape
    bt = _device_tensor(block_tables, "block_tables", dev, i32)
    sl = _device_tensor(seq_lens, "seq_lens", dev, i32, (n,))
    nl = _device_tensor(new_lens, "new_lens", dev, i32, (n,))
    nb = _device_tensor(n_blocks, "n_blocks", dev, i32, (n,))
    fl = _device_tensor(free_list, "free_list", dev, i32)
    fc = _device_tensor(free_count, "free_count", dev, i32, (1,))
    s, ctx = _run_on(stream, dev, (bt, sl, nl, nb, fl, fc))
    with ctx:
        tables = torch.empty((n, width), dtype=i32, device=dev)
        # the small arrays share one allocation
        small = torch.empty(3 * n + 3 + 2 * max_tokens, dtype=i32, device=dev)
        r = StepTables(tables, *small.split((n, 1, n, n + 1, max_tokens, max_tokens, 1)))
        p = _dev_ptr(small)
        ctx_at = p + 4 * n + 4
        pos_at = ctx_at + 8 * n + 4
        slot_at = pos_at + 4 * max_tokens
        check(lib().pkv_step_tables(
            block_size, num_blocks, _dev_ptr(sl), _dev_ptr(nl), n, _dev_ptr(bt), _dev_ptr(nb),
            width, _dev_ptr(fl), fl.numel(), _dev_ptr(fc), max_tokens, _dev_ptr(tables), p,
            p + 4 * n, ctx_at, ctx_at + 4 * n, pos_at, slot_at, slot_at + 4 * max_tokens, s), None)
    return r


def verify_drafts(target_logits, draft_tokens, cu_drafts, uniforms, final_uniforms,
                  draft_logits=None, temperatures=None, stream=None):
    """Keeps the drafted tokens that the target's distribution keeps and draws
    the token after them (pkv_verify_drafts), from given random numbers.
    target_logits: (drafts + batch, vocab) f32/f16/bf16, request b's rows (one
    per draft and one after the last) at cu_drafts[b] + b; draft_tokens:
    (drafts,) int32; cu_drafts: (batch + 1,) int32; uniforms: (drafts,) and
    final_uniforms: (batch,) float32 in [0, 1); draft_logits: (drafts, vocab)
    f32/f16/bf16, or None for drafts without a distribution; temperatures:
    (batch,) float32, or None (all greedy; so is one that is not positive
    or not finite).  Both logits have unit
    stride along vocab.  Draft i is kept while u_i q_i(d_i) < p_i(d_i); the next
    token comes from max(p - q, 0) of the first one that is not, or from p
    after the last.  Nothing synchronises.  Returns (tokens, accepted):
    (drafts + batch,) int32 with a request's kept drafts, next token and then
    -1 at cu_drafts[b] + b, and (batch,) int32 with the number of kept drafts.
    cu_drafts runs from 0 to drafts; what no request covers is not written."""
    import torch
    if not isinstance(target_logits, torch.Tensor) or not target_logits.is_cuda:
        raise ValueError("target_logits must be a device tensor")
    dev, i32, f32 = target_logits.device, torch.int32, torch.float32
    total, batch = draft_tokens.numel(), final_uniforms.numel()
    for t, name, rows in ((target_logits, "target_logits", total + batch),
                          (draft_logits, "draft_logits", total)):
        if t is None:
            continue
        if t.device != dev or t.dim() != 2 or t.shape[0] != rows or \
                t.shape[1] != target_logits.shape[1] or \
                (t.numel() and t.shape[1] > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be ({rows}, vocab) on {dev} with unit stride along "
                             "vocab")
    vocab = target_logits.shape[1]
    dt = _device_tensor(draft_tokens, "draft_tokens", dev, i32, (total,))
    cu = _device_tensor(cu_drafts, "cu_drafts", dev, i32, (batch + 1,))
    u = _device_tensor(uniforms, "uniforms", dev, f32, (total,))
    uf = _device_tensor(final_uniforms, "final_uniforms", dev, f32, (batch,))
    tp = None
    if temperatures is not None:
        tp = _device_tensor(temperatures, "temperatures", dev, f32, (batch,))
    has_draft = draft_logits is not None and total > 0
    s, ctx = _run_on(stream, dev, (target_logits, draft_logits, dt, cu, u, uf, tp))
    with ctx:
        tokens, accepted = torch.empty(total + 2 * batch, dtype=i32, device=dev).split(
            (total + batch, batch))
        need = lib().pkv_verify_workspace_bytes(batch, total, vocab, has_draft)
        ws = _workspace(need, dev)
        check(lib().pkv_verify_drafts(
            _dev_ptr(target_logits), pkv_dtype(target_logits.dtype),
            max(target_logits.stride(0), vocab) if total + batch <= 1 else target_logits.stride(0),
            _dev_ptr(draft_logits) if has_draft else None,
            pkv_dtype(draft_logits.dtype) if has_draft else F32,
            (max(draft_logits.stride(0), vocab) if total <= 1 else draft_logits.stride(0))
            if has_draft else 0,
            _dev_ptr(dt), _dev_ptr(cu), batch, total, vocab, _dev_ptr(u), _dev_ptr(uf),
            _dev_ptr(tp) if tp is not None else None, _dev_ptr(tokens), _dev_ptr(accepted),
            _dev_ptr(ws), need, s), None)
    return tokens, accepted


class Rope:
    """The reference's Rope (rope.rs:6-33): cos/sin tables in device memory;
    apply() is apply_rope (rope.rs:38-42) with per-token positions."""

    def __init__(self, rope_dim: int, freq_base: float, max_seq: int, device: int = 0) -> None:
        import torch
        h = ctypes.c_void_p()
        check(lib().pkv_rope_create(ctypes.byref(h), rope_dim, freq_base, max_seq, device), None)
        self._h = h
        self.rope_dim, self.freq_base, self.max_seq = rope_dim, freq_base, max_seq
        self.device = torch.device("cuda", device)

    @property
    def handle(self):
        return self._h

    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            lib().pkv_rope_destroy(h)
            self._h = None

    def __del__(self, _finalizing=sys.is_finalizing) -> None:
        # at interpreter exit the module's globals may already be gone; the
        # process end releases the device memory
        if not _finalizing():
            self.close()

    def apply(self, x, positions, out_dtype=None, out=None, stream=None):
        """x: (n_tokens, n_head, rope_dim) f32/f16/bf16 on the device;
        positions: (n_tokens,) int32.  Returns the rotated rows."""
        import torch
        if x.dim() != 3 or x.shape[2] != self.rope_dim:
            raise ValueError(f"x must be (n, heads, {self.rope_dim})")
        xx = x.contiguous()
        if out is None:
            out = torch.empty(xx.shape, dtype=out_dtype or xx.dtype, device=xx.device)
        pos = _i32(positions, xx.device)
        check(lib().pkv_rope_apply(self._h, _dev_ptr(xx), pkv_dtype(xx.dtype), _dev_ptr(out),
                                   pkv_dtype(out.dtype), _dev_ptr(pos), xx.shape[0],
                                   xx.shape[1], _stream_ptr(stream)), None)
        return out

    def check(self) -> None:
        check(lib().pkv_rope_check(self._h), None)


class PagedKvCache:
    """K/V pools of every layer on one GPU (the reference's Vec<KvPool>,
    engine.rs:70-72; KvPool::new, attention.rs:39-55).  Zero-initialised,
    layout [layer][K|V][num_blocks][block_size][n_kv_head][head_dim]."""

    def __init__(self, n_layers: int, num_blocks: int, block_size: int, n_kv_head: int,
                 head_dim: int, dtype=None, device: int = 0) -> None:
        import torch
        if dtype is None:
            dtype = torch.float32
        self.dtype = dtype
        self.n_layers, self.num_blocks, self.block_size = n_layers, num_blocks, block_size
        self.n_kv_head, self.head_dim, self.device_index = n_kv_head, head_dim, device
        self.device = torch.device("cuda", device)
        h = ctypes.c_void_p()
        rc = lib().pkv_pool_create(ctypes.byref(h), n_layers, num_blocks, block_size,
                                   n_kv_head, head_dim, pkv_dtype(dtype), device)
        check(rc, None)
        self._h = h

    @property
    def handle(self):
        return self._h

    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            lib().pkv_pool_destroy(h)
            self._h = None

    def __del__(self, _finalizing=sys.is_finalizing) -> None:
        # at interpreter exit the module's globals may already be gone; the
        # process end releases the device memory
        if not _finalizing():
            self.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    def layer(self, l: int) -> "KvPool":
        if not 0 <= l < self.n_layers:
            raise IndexError(l)
        return KvPool(self, l)

    @property
    def layer_bytes(self) -> int:
        return int(lib().pkv_pool_layer_bytes(self._h))

    @property
    def block_bytes(self) -> int:
        return self.layer_bytes // self.num_blocks

    def fill_normal(self, seed: int, stream=None) -> None:
        check(lib().pkv_pool_fill_normal(self._h, seed, _stream_ptr(stream)), self._h)

    def verify_normal(self, seed: int, blocks, origin, stream=None) -> int:
        """16-byte chunks of blocks[i] (all layers, K and V) that differ from
        what fill_normal(seed) wrote into block origin[i] (synchronous)."""
        b = _i32(blocks, self.device)
        o = _i32(origin, self.device)
        if b.numel() != o.numel():
            raise ValueError("blocks and origin must have the same length")
        n = ctypes.c_uint64()
        check(lib().pkv_pool_verify_normal(self._h, seed, _dev_ptr(b), _dev_ptr(o), b.numel(),
                                           ctypes.byref(n), _stream_ptr(stream)), self._h)
        return int(n.value)

    def read_blocks(self, blocks, out=None, stream=None):
        """Reads every byte of blocks[i] (all layers, K and V) on the device
        and adds their 32-bit words (mod 2^64) into out, a device int64
        tensor of one element holding the unsigned sum's bits (zeroed here
        unless given); returns out.  Asynchronous."""
        import torch
        b = _i32(blocks, self.device)
        if out is None:
            out = torch.zeros(1, dtype=torch.int64, device=self.device)
        if out.dtype != torch.int64 or out.numel() < 1 or not out.is_cuda:
            raise ValueError("out must be a device int64 tensor")
        check(lib().pkv_pool_read_blocks(self._h, _dev_ptr(b), b.numel(), _dev_ptr(out),
                                         _stream_ptr(stream)), self._h)
        return out

    def copy_blocks(self, src, dst, stream=None) -> None:
        """Copy-on-write: block dst[i] <- src[i] in every layer, K and V."""
        s = _i32(src, self.device)
        d = _i32(dst, self.device)
        if s.numel() != d.numel():
            raise ValueError("src/dst length mismatch")
        check(lib().pkv_copy_blocks(self._h, _dev_ptr(s), _dev_ptr(d), s.numel(),
                                    _stream_ptr(stream)), self._h)

    def compact(self, src: Sequence[int], dst: Sequence[int], stream=None) -> None:
        """In-place block moves src[i] -> dst[i] (sets may overlap)."""
        import numpy as np
        s = np.ascontiguousarray(src, dtype=np.int32)
        d = np.ascontiguousarray(dst, dtype=np.int32)
        if s.size != d.size:
            raise ValueError("src/dst length mismatch")
        P = ctypes.POINTER(ctypes.c_int32)
        check(lib().pkv_compact(self._h, s.ctypes.data_as(P), d.ctypes.data_as(P), s.size,
                                _stream_ptr(stream)), self._h)

    def check(self) -> None:
        """Raise if a kernel met an out-of-range id or length since last check."""
        check(lib().pkv_pool_check(self._h), self._h)

    def profile(self, enable: bool) -> None:
        """Record HIP events around every decode call's main kernel."""
        check(lib().pkv_pool_profile(self._h, 1 if enable else 0), self._h)

    def profile_read(self) -> tuple[float, int]:
        """(summed main-kernel ms, launches) since the last read."""
        ms = ctypes.c_double()
        n = ctypes.c_int()
        check(lib().pkv_pool_profile_read(self._h, ctypes.byref(ms), ctypes.byref(n)), self._h)
        return float(ms.value), int(n.value)

    def decode_workspace_bytes(self, batch: int, n_head: int, max_context_len: int) -> int:
        return int(lib().pkv_decode_workspace_bytes(self._h, batch, n_head, max_context_len))

    def reserve_decode(self, batch: int, n_head: int, max_context_len: int) -> None:
        check(lib().pkv_pool_reserve_decode(self._h, batch, n_head, max_context_len), self._h)

    def prefill_workspace_bytes(self, n_seqs: int, n_head: int, max_q_len: int,
                                max_context_len: int) -> int:
        return int(lib().pkv_prefill_workspace_bytes(self._h, n_seqs, n_head, max_q_len,
                                                     max_context_len))

    def reserve_prefill(self, n_seqs: int, n_head: int, max_q_len: int,
                        max_context_len: int) -> None:
        check(lib().pkv_pool_reserve_prefill(self._h, n_seqs, n_head, max_q_len,
                                             max_context_len), self._h)

    # raw byte access (synchronous), for tests and checkpoints
    def read_bytes(self, layer: int, which: int, offset: int = 0, nbytes: int | None = None):
        import numpy as np
        if nbytes is None:
            nbytes = self.layer_bytes - offset
        buf = np.empty(nbytes, dtype=np.uint8)
        check(lib().pkv_pool_read(self._h, layer, which, offset, nbytes, buf.ctypes.data), self._h)
        return buf

    def write_bytes(self, layer: int, which: int, data, offset: int = 0) -> None:
        import numpy as np
        a = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        check(lib().pkv_pool_write(self._h, layer, which, offset, a.ctypes.data, a.size), self._h)


class KvPool:
    """One layer of a PagedKvCache: the reference's KvPool (attention.rs:30-98)."""

    def __init__(self, cache: PagedKvCache, layer: int) -> None:
        self.cache = cache
        self.layer_index = layer

    @property
    def _h(self):
        return self.cache.handle

    # -- KvPool::write (attention.rs:57-83) --------------------------------
    def write(self, alloc: BlockAllocator, table: BlockTable, start_pos: int, k, v,
              stream=None) -> None:
        n_new = int(k.shape[0])
        slots = [alloc.slot(table, start_pos + i) for i in range(n_new)]
        self.append(k, v, slots, stream)

    def append(self, k, v, slot_mapping, stream=None) -> None:
        """Scatter k, v (n, n_kv, hd) to the given slots (int32, -1 = skip)."""
        c = self.cache
        self._check_rows(k, "k")
        self._check_rows(v, "v")
        sm = _i32(slot_mapping, c.device)
        if sm.numel() != k.shape[0] or v.shape[0] != k.shape[0]:
            raise ValueError("slot_mapping / k / v lengths differ")
        check(lib().pkv_append(self._h, self.layer_index, _dev_ptr(k), _dev_ptr(v),
                               _dev_ptr(sm), k.shape[0], _stream_ptr(stream)), self._h)

    def append_rope(self, rope: "Rope", k, v, slot_mapping, positions, q=None, q_out=None,
                    stream=None):
        """prefill_seq's glue (transformer.rs:160-174) in one launch: rotate k
        (n, n_kv, hd) by `positions`, store it and v at `slot_mapping`, and,
        with q (n, H, hd), return q rotated into the pool dtype (into q_out if
        given).  k, v, q share one dtype: float32 or the pool dtype."""
        import torch
        c = self.cache
        n = int(k.shape[0])
        if q is not None and q.dtype != k.dtype:
            raise TypeError("q must have k's dtype")
        if k.dtype not in (torch.float32, c.dtype) or v.dtype != k.dtype:
            raise TypeError("k and v must be float32 or the pool dtype, and equal")
        for t, name in ((k, "k"), (v, "v")):
            if t.shape != (n, c.n_kv_head, c.head_dim) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous ({n}, {c.n_kv_head}, {c.head_dim})")
        sm = _i32(slot_mapping, c.device)
        pos = _i32(positions, c.device)
        if sm.numel() != n or pos.numel() != n:
            raise ValueError("slot_mapping / positions / k lengths differ")
        H = 0
        if q is not None:
            if q.dim() != 3 or q.shape[0] != n or q.shape[2] != c.head_dim:
                raise ValueError(f"q must be ({n}, H, {c.head_dim})")
            q = q.contiguous()
            H = int(q.shape[1])
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=c.dtype, device=c.device)
            if q_out.dtype != c.dtype or q_out.shape != q.shape or not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous, q's shape, in the pool dtype")
        check(lib().pkv_append_rope(
            self._h, self.layer_index, rope.handle, _dev_ptr(pos), pkv_dtype(k.dtype),
            _dev_ptr(k), _dev_ptr(v), _dev_ptr(sm), n,
            _dev_ptr(q) if q is not None else None,
            _dev_ptr(q_out) if q is not None else None, H, _stream_ptr(stream)), self._h)
        return q_out if q is not None else None

    # -- KvPool::gather_seq (attention.rs:85-97) ----------------------------
    def gather_seq(self, table, length: int, stream=None):
        import torch
        c = self.cache
        blocks = table.blocks if isinstance(table, BlockTable) else list(table)
        need = -(-length // c.block_size)
        if need > len(blocks):
            raise IndexError("length beyond the block table")
        tb = _i32(blocks[:max(need, 1)] if blocks else [0], c.device)
        ok = torch.empty((length, c.n_kv_head, c.head_dim), dtype=c.dtype, device=c.device)
        ov = torch.empty_like(ok)
        check(lib().pkv_gather_seq(self._h, self.layer_index, _dev_ptr(tb), length,
                                   _dev_ptr(ok), _dev_ptr(ov), _stream_ptr(stream)), self._h)
        return ok, ov

    def gather_varlen(self, block_tables, lengths, stream=None):
        """Several sequences' K/V in one launch: rows of sequence b at
        cu[b] .. cu[b+1]-1 of the returned (total, n_kv, hd) K and V, where
        cu = [0, cumsum(lengths)]; returns (k, v, cu) with cu on the device."""
        import numpy as np
        import torch
        c = self.cache
        lens = np.asarray(lengths, np.int64)
        cu_np = np.zeros(lens.size + 1, np.int32)
        cu_np[1:] = np.cumsum(lens)
        total = int(cu_np[-1])
        bt = _i32(block_tables, c.device)
        cu = torch.from_numpy(cu_np).to(c.device)
        ok = torch.empty((total, c.n_kv_head, c.head_dim), dtype=c.dtype, device=c.device)
        ov = torch.empty_like(ok)
        if total:
            check(lib().pkv_gather_varlen(self._h, self.layer_index, _dev_ptr(bt), bt.shape[1],
                                          _dev_ptr(cu), lens.size, total, _dev_ptr(ok),
                                          _dev_ptr(ov), _stream_ptr(stream)), self._h)
        return ok, ov, cu

    # -- decode attention ---------------------------------------------------
    def decode_attention(self, q, block_tables, context_lens, max_context_len: int | None = None,
                         k_new=None, v_new=None, scale: float | None = None, out_dtype=None,
                         out=None, stream=None, rope: "Rope | None" = None, positions=None):
        """q: (B, H, hd); block_tables: (B, max_nb) int32 device; context_lens:
        (B,) int32 device = keys attended (seq_lens + 1).  With k_new/v_new
        (B, n_kv, hd) the new token is stored at position context_lens-1 first.
        With `rope`, q and k_new are the projections before rotation (f32 or
        the pool dtype) and the kernel applies the rotary embedding at
        `positions` (default context_lens - 1).  Given, `positions` ((B,)
        int32 device) also bound the keys attended: k <= positions[b]
        (build_mask's second bound; pkv_decode_attention_positions without
        rope).  Returns (B, H*hd)."""
        if rope is not None:
            return self._decode_attention_rope(q, block_tables, context_lens, max_context_len,
                                               k_new, v_new, scale, out_dtype, out, stream,
                                               rope, positions)
        import torch
        c = self.cache
        B, H, hd = q.shape
        if hd != c.head_dim:
            raise ValueError("head_dim mismatch")
        if out_dtype is None:
            out_dtype = q.dtype
        if scale is None:
            scale = 1.0 / math.sqrt(hd)
        bt = _i32(block_tables, c.device)
        cl = _i32(context_lens, c.device)
        if max_context_len is None:
            max_context_len = int(cl.max().item()) if B else 1
        if out is None:
            out = torch.empty((B, H * hd), dtype=out_dtype, device=c.device)
        if k_new is not None:
            self._check_rows(k_new, "k_new")
            self._check_rows(v_new, "v_new")
        qq = q.contiguous()
        if qq.dtype != c.dtype:
            raise TypeError("q must have the pool dtype")
        kv = (_dev_ptr(k_new) if k_new is not None else None,
              _dev_ptr(v_new) if v_new is not None else None, _stream_ptr(stream))
        if positions is not None:
            pos = _i32(positions, c.device)
            check(lib().pkv_decode_attention_positions(
                self._h, self.layer_index, _dev_ptr(qq), _dev_ptr(out), pkv_dtype(out.dtype),
                _dev_ptr(bt), bt.shape[1], _dev_ptr(cl), _dev_ptr(pos), int(max_context_len), B,
                H, float(scale), *kv), self._h)
            return out
        check(lib().pkv_decode_attention(
            self._h, self.layer_index, _dev_ptr(qq), _dev_ptr(out), pkv_dtype(out.dtype),
            _dev_ptr(bt), bt.shape[1], _dev_ptr(cl), int(max_context_len), B, H, float(scale),
            *kv), self._h)
        return out

    def _decode_attention_rope(self, q, block_tables, context_lens, max_context_len, k_new,
                               v_new, scale, out_dtype, out, stream, rope, positions):
        import torch
        c = self.cache
        B, H, hd = q.shape
        if hd != c.head_dim:
            raise ValueError("head_dim mismatch")
        if q.dtype not in (torch.float32, c.dtype):
            raise TypeError("q must be float32 or the pool dtype")
        for t, name in ((k_new, "k_new"), (v_new, "v_new")):
            if t is not None and (t.dtype != q.dtype or t.shape != (B, c.n_kv_head, hd)):
                raise ValueError(f"{name} must be ({B}, {c.n_kv_head}, {hd}) in q's dtype")
        if scale is None:
            scale = 1.0 / math.sqrt(hd)
        bt = _i32(block_tables, c.device)
        cl = _i32(context_lens, c.device)
        if max_context_len is None:
            max_context_len = int(cl.max().item()) if B else 1
        if out is None:
            out = torch.empty((B, H * hd), dtype=out_dtype or c.dtype, device=c.device)
        pos = _i32(positions, c.device) if positions is not None else None
        qq = q.contiguous()
        kk = k_new.contiguous() if k_new is not None else None
        vv = v_new.contiguous() if v_new is not None else None
        check(lib().pkv_decode_attention_rope(
            self._h, self.layer_index, rope.handle, _dev_ptr(pos) if pos is not None else None,
            pkv_dtype(qq.dtype), _dev_ptr(qq), _dev_ptr(out), pkv_dtype(out.dtype), _dev_ptr(bt),
            bt.shape[1], _dev_ptr(cl), int(max_context_len), B, H, float(scale),
            _dev_ptr(kk) if kk is not None else None, _dev_ptr(vv) if vv is not None else None,
            _stream_ptr(stream)), self._h)
        return out

    # -- chunked prefill attention -------------------------------------------
    def prefill_attention(self, q, cu_q_lens, context_lens, block_tables, max_q_len: int,
                          max_context_len: int, scale: float | None = None, out_dtype=None,
                          out=None, stream=None, k_new=None, v_new=None):
        """Causal attention of prompt chunks over prior context + chunk.  With
        k_new / v_new (total_q, n_kv, hd), the chunk's K/V are stored in the
        same launch (pkv_prefill_attention_append); without, they must
        already be in the pool."""
        import torch
        c = self.cache
        T, H, hd = q.shape
        if out_dtype is None:
            out_dtype = q.dtype
        if scale is None:
            scale = 1.0 / math.sqrt(hd)
        cu = _i32(cu_q_lens, c.device)
        cl = _i32(context_lens, c.device)
        bt = _i32(block_tables, c.device)
        if out is None:
            out = torch.empty((T, H * hd), dtype=out_dtype, device=c.device)
        args = [self._h, self.layer_index, _dev_ptr(q.contiguous()), _dev_ptr(out),
                pkv_dtype(out.dtype), _dev_ptr(cu), _dev_ptr(cl), _dev_ptr(bt), bt.shape[1],
                cl.numel(), int(max_q_len), int(max_context_len), H, float(scale)]
        if k_new is not None or v_new is not None:
            self._check_rows(k_new, "k_new")
            self._check_rows(v_new, "v_new")
            check(lib().pkv_prefill_attention_append(*args, _dev_ptr(k_new), _dev_ptr(v_new),
                                                     _stream_ptr(stream)), self._h)
        else:
            check(lib().pkv_prefill_attention(*args, _stream_ptr(stream)), self._h)
        return out

    # -- a layer's mixed batch -------------------------------------------------
    def mixed_attention(self, prefill: dict, decode: dict, scale: float | None = None,
                        stream=None):
        """pkv_mixed_attention: the prefill batch (keys of prefill_attention:
        q, cu_q_lens, context_lens, block_tables, max_q_len, max_context_len,
        optional k_new, v_new, out_dtype, out) and the decode batch (keys of
        decode_attention: q, block_tables, context_lens, optional
        max_context_len, k_new, v_new, out_dtype, out) of one layer in one
        call; results identical to the two calls.  Returns (prefill out,
        decode out)."""
        import torch
        c = self.cache
        pq, dq = prefill["q"].contiguous(), decode["q"].contiguous()
        H, hd = pq.shape[1], pq.shape[2]
        if dq.shape[1:] != (H, hd) or hd != c.head_dim:
            raise ValueError("prefill and decode q must be (n, n_head, head_dim) of the pool")
        if pq.dtype != c.dtype or dq.dtype != c.dtype:
            raise TypeError("q must have the pool dtype")
        if scale is None:
            scale = 1.0 / math.sqrt(hd)
        keep = []  # tensors the structs point into, alive until the call returns

        def dev(t):
            keep.append(t)
            return _dev_ptr(t)

        rows = {}
        for side, d in (("prefill", prefill), ("decode", decode)):
            for key in ("k_new", "v_new"):
                if d.get(key) is not None:
                    self._check_rows(d[key], key)
            n = (d["q"].shape[0])
            out = d.get("out")
            if out is None:
                out = torch.empty((n, H * hd), dtype=d.get("out_dtype") or c.dtype,
                                  device=c.device)
            rows[side] = out
        pcu = _i32(prefill["cu_q_lens"], c.device)
        pcl = _i32(prefill["context_lens"], c.device)
        pbt = _i32(prefill["block_tables"], c.device)
        dcl = _i32(decode["context_lens"], c.device)
        dbt = _i32(decode["block_tables"], c.device)
        dmax = decode.get("max_context_len")
        if dmax is None:
            dmax = int(dcl.max().item()) if dcl.numel() else 1
        pk, pv = prefill.get("k_new"), prefill.get("v_new")
        dk, dv = decode.get("k_new"), decode.get("v_new")
        pb = _lib.PrefillBatch(dev(pq), dev(rows["prefill"]), pkv_dtype(rows["prefill"].dtype),
                               dev(pcu), dev(pcl), dev(pbt), pbt.shape[1], pcl.numel(),
                               int(prefill["max_q_len"]), int(prefill["max_context_len"]),
                               dev(pk) if pk is not None else None,
                               dev(pv) if pv is not None else None)
        db = _lib.DecodeBatch(dev(dq), dev(rows["decode"]), pkv_dtype(rows["decode"].dtype),
                              dev(dbt), dbt.shape[1], dev(dcl), int(dmax), dcl.numel(),
                              dev(dk) if dk is not None else None,
                              dev(dv) if dv is not None else None)
        check(lib().pkv_mixed_attention(self._h, self.layer_index, ctypes.byref(pb),
                                        ctypes.byref(db), H, float(scale),
                                        _stream_ptr(stream)), self._h)
        return rows["prefill"], rows["decode"]

    # -- attention over chosen blocks -------------------------------------------
    def new_key_bounds(self):
        """Zeroed key bounds of one layer: (num_blocks, n_kv, 2, hd) in the pool
        dtype, the smallest and the largest key element of each block."""
        import torch
        c = self.cache
        return torch.zeros((c.num_blocks, c.n_kv_head, 2, c.head_dim), dtype=c.dtype,
                           device=c.device)

    def _check_bounds(self, bounds) -> None:
        c = self.cache
        shape = (c.num_blocks, c.n_kv_head, 2, c.head_dim)
        if _device_tensor(bounds, "bounds", c.device, c.dtype, shape) is not bounds:
            raise ValueError("bounds must be contiguous")

    def update_key_bounds(self, bounds, block_tables, context_lens, first_positions=None,
                          max_new_len: int | None = None, stream=None):
        """Brings `bounds` (new_key_bounds) up to date for every block that holds
        a position from first_positions[s] (None: 0) to context_lens[s] - 1 of
        a sequence (pkv_key_bounds).  block_tables: (n, width) int32;
        context_lens, first_positions: (n,) int32; max_new_len: host bound of
        their difference (None: what the tables hold).  Returns bounds."""
        c = self.cache
        self._check_bounds(bounds)
        bt, cl = _i32_on(block_tables, c.device), _i32_on(context_lens, c.device)
        fp = _i32_on(first_positions, c.device) if first_positions is not None else None
        n = cl.numel()
        if bt.dim() != 2 or bt.shape[0] != n or (fp is not None and fp.numel() != n):
            raise ValueError("block_tables must be (n, width), context_lens and "
                             "first_positions (n,)")
        if max_new_len is None:
            max_new_len = bt.shape[1] * c.block_size
        s, ctx = _run_on(stream, c.device, (bounds, bt, cl, fp))
        with ctx:
            check(lib().pkv_key_bounds(
                self._h, self.layer_index, _dev_ptr(bounds), _dev_ptr(bt), bt.shape[1],
                _dev_ptr(fp) if fp is not None else None, _dev_ptr(cl), n, int(max_new_len), s),
                self._h)
        return bounds

    def _rows(self, q, block_tables, context_lens, cu_q_lens, max_q_len):
        """Checked row arguments of select_blocks and sparse_attention."""
        import torch
        c = self.cache
        if q.device != c.device or q.dim() != 3 or q.shape[2] != c.head_dim:
            raise ValueError(f"q must be (rows, n_head, {c.head_dim}) on {c.device}")
        if q.dtype != c.dtype:
            raise TypeError("q must have the pool dtype")
        bt, cl = _i32_on(block_tables, c.device), _i32_on(context_lens, c.device)
        cu = _i32_on(cu_q_lens, c.device) if cu_q_lens is not None else None
        n, rows = cl.numel(), q.shape[0]
        if bt.dim() != 2 or bt.shape[0] != n:
            raise ValueError("block_tables must be (n, width), context_lens (n,)")
        if cu is not None and cu.numel() != n + 1:
            raise ValueError("cu_q_lens must be (n + 1,)")
        if cu is None and rows != n:
            raise ValueError("without cu_q_lens q has one row per sequence")
        if max_q_len is None:
            max_q_len = 1
            if cu is not None and getattr(cu_q_lens, "is_cuda", False):
                max_q_len = max(rows, 1)  # (a bound without a synchronisation)
            elif cu is not None and n:
                max_q_len = max(int(torch.as_tensor(cu_q_lens, dtype=torch.int64).diff().max()), 1)
        return q.contiguous(), bt, cl, cu, n, rows, int(max_q_len)

    def select_blocks(self, q, bounds, block_tables, context_lens, top_blocks: int,
                      first_blocks: int = 1, last_blocks: int = 1, cu_q_lens=None,
                      max_q_len: int | None = None, max_context_len: int | None = None, out=None,
                      stream=None):
        """The blocks that each query row attends, per kv head (pkv_select_blocks):
        the first and last ones of its context and, of those between, the ones
        whose `bounds` promise the group's heads the largest score, top_blocks in
        all.  q: (rows, H, hd) in the pool dtype, as the attention will get it;
        context_lens: (n,) int32; block_tables: (n, width) int32; cu_q_lens: (n + 1,)
        int32 (None: one row per sequence), row i of a chunk of m rows having
        the keys up to position context_lens - m + i.  max_context_len: host bound
        (None: what the tables hold).  max_q_len: host bound of the chunks (None:
        the longest one if cu_q_lens is on the host, else all rows).  The launch
        has n * max_q_len row places, so a batch whose cu_q_lens is on the device
        should pass it: many requests under a loose bound cost time or are
        refused.  Returns (rows, n_kv, top_blocks) int32, ascending indexes into
        the sequence's row of block_tables, then -1 (into `out` if given).  Rows of
        no sequence and those of a chunk beyond max_q_len are not written: as they
        were in `out`, uninitialised without it."""
        import torch
        c = self.cache
        self._check_bounds(bounds)
        qq, bt, cl, cu, n, rows, mq = self._rows(q, block_tables, context_lens, cu_q_lens,
                                                 max_q_len)
        H = qq.shape[1]
        if max_context_len is None:
            max_context_len = bt.shape[1] * c.block_size
        shape = (rows, c.n_kv_head, top_blocks)
        if out is not None and _device_tensor(out, "out", c.device, torch.int32, shape) is not out:
            raise ValueError("out must be contiguous")
        s, ctx = _run_on(stream, c.device, (qq, bounds, bt, cl, cu, out))
        with ctx:
            if out is None:
                out = torch.empty(shape, dtype=torch.int32, device=c.device)
            need = lib().pkv_select_workspace_bytes(self._h, n, rows, mq, int(max_context_len),
                                                    bt.shape[1], H)
            ws = _workspace(need, c.device)
            check(lib().pkv_select_blocks(
                self._h, _dev_ptr(qq), _dev_ptr(bounds), _dev_ptr(out), int(top_blocks),
                int(first_blocks), int(last_blocks), _dev_ptr(cu) if cu is not None else None,
                _dev_ptr(cl), _dev_ptr(bt), bt.shape[1], n, rows, mq, int(max_context_len), H,
                _dev_ptr(ws), need, s), self._h)
        return out

    def sparse_attention(self, q, blocks, block_tables, context_lens, cu_q_lens=None,
                         max_q_len: int | None = None, scale: float | None = None, out_dtype=None,
                         out=None, stream=None):
        """Attention of each query row over the keys of its listed blocks
        (pkv_sparse_attention).  blocks: (rows, n_kv, top) int32, as select_blocks
        returns them (any order, distinct; negative entries are skipped); the
        other arguments as select_blocks' (whether max_q_len is 1 or more also
        decides how lists are cut, so it may change last bits).  The rows' keys
        are in the pool already.  Returns (rows, H * hd); a row without keys is
        zero, one that select_blocks would not write is not written."""
        import torch
        c = self.cache
        qq, bt, cl, cu, n, rows, mq = self._rows(q, block_tables, context_lens, cu_q_lens,
                                                 max_q_len)
        H, hd = qq.shape[1], qq.shape[2]
        if blocks.dim() != 3 or blocks.shape[:2] != (rows, c.n_kv_head):
            raise ValueError(f"blocks must be ({rows}, {c.n_kv_head}, top)")
        bl = _device_tensor(blocks, "blocks", c.device, torch.int32)
        if scale is None:
            scale = 1.0 / math.sqrt(hd)
        if out is not None and (out.device != c.device or out.shape != (rows, H * hd)
                                or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous ({rows}, {H * hd}) on {c.device}")
        s, ctx = _run_on(stream, c.device, (qq, bl, bt, cl, cu, out))
        with ctx:
            if out is None:
                out = torch.empty((rows, H * hd), dtype=out_dtype or c.dtype, device=c.device)
            need = lib().pkv_sparse_workspace_bytes(self._h, rows, H, bl.shape[2])
            ws = _workspace(need, c.device) if need else None
            check(lib().pkv_sparse_attention(
                self._h, self.layer_index, _dev_ptr(qq), _dev_ptr(out), pkv_dtype(out.dtype),
                _dev_ptr(bl), bl.shape[2], _dev_ptr(cu) if cu is not None else None,
                _dev_ptr(cl), _dev_ptr(bt), bt.shape[1], n, rows, mq, H, float(scale),
                _dev_ptr(ws) if need else None, need, s), self._h)
        return out

    def _check_rows(self, t, name: str) -> None:
        c = self.cache
        if t.dtype != c.dtype:
            raise TypeError(f"{name} must have the pool dtype {c.dtype}")
        if t.dim() != 3 or t.shape[1] != c.n_kv_head or t.shape[2] != c.head_dim:
            raise ValueError(f"{name} must be (n, {c.n_kv_head}, {c.head_dim})")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
