"""Host-side mirror of molla's device entry points, over the C ABI.

Mirrors src/molla/nn/gpu.mojo (device_matvec_into :2148, device_matmul_into
:2945, device_matvec :3112), src/molla/nn/gpu_ops.mojo (rms_norm, rope,
store_kv, attend, argmax) and src/molla/nn/tensor.mojo (the Tensor view):
same names, same argument meaning, same refusals raised before anything is
queued.  Device memory and streams come from PyTorch (ROCm); the arithmetic is
all in libmolla_mi.so.  There is no CPU fallback: without the library or a
GPU every call raises.
"""

from __future__ import annotations

import ctypes
import functools

import numpy as np
import torch

from ._lib import MiError, MiExperts, MiLayerDesc, MiQk, MiTree, MiWeight, check, lib

# ggml type numbers, src/molla/nn/quant.mojo:47-57
Q_F32, Q_F16, Q_Q4_0, Q_Q4_1, Q_Q5_0, Q_Q5_1, Q_Q8_0, Q_Q4_K, Q_Q5_K, Q_Q6_K = 0, 1, 2, 3, 6, 7, 8, 12, 13, 14
KIND_NAMES = {0: "F32", 1: "F16", 2: "Q4_0", 3: "Q4_1", 6: "Q5_0", 7: "Q5_1", 8: "Q8_0", 12: "Q4_K", 13: "Q5_K",
              14: "Q6_K"}
# epilogues, src/molla/nn/gpu.mojo:781-803
EPI_NONE, EPI_BIAS, EPI_ADD, EPI_GLU, ACT_BIT = 0, 1, 2, 4, 8

WHERE_DEVICE = 2


def block_elements(kind: int) -> int:
    return lib().mi_block_elements(kind)


def block_bytes(kind: int) -> int:
    return lib().mi_block_bytes(kind)


class Tensor:
    """A view of a packed weight that owns nothing (tensor.mojo:66-121).

    `cols` is the fast axis (ggml order, tensor.mojo:15-19): a (rows x cols)
    matrix of `kind` blocks, rows back to back.  `address` is a device
    pointer; `keep` holds whatever owns the memory (a torch tensor).
    """

    def __init__(self, address: int, kind: int, cols: int, rows: int, keep=None):
        self.address = int(address)
        self.kind = kind
        self.cols = cols
        self.rows = rows
        self.place = WHERE_DEVICE
        self.keep = keep

    @staticmethod
    def from_bytes(blob, kind: int, cols: int, rows: int, device="cuda") -> "Tensor":
        """Upload raw GGUF bytes (numpy uint8 or a torch uint8 tensor) to the device."""
        t = torch.as_tensor(blob, dtype=torch.uint8) if not isinstance(blob, torch.Tensor) else blob
        t = t.to(device).contiguous()
        want = rows * row_bytes(kind, cols)
        if t.numel() != want:
            raise ValueError(f"{rows} rows of {cols} type-{kind} values take {want} bytes, got {t.numel()}")
        return Tensor(t.data_ptr(), kind, cols, rows, keep=t)

    def row_bytes(self) -> int:
        return row_bytes(self.kind, self.cols)

    def elements(self) -> int:
        return self.rows * self.cols

    def weight(self) -> MiWeight:
        return MiWeight(self.address, self.kind, self.rows, self.cols, self.row_bytes())


# (a size of its two numbers alone; asked of the library each time it is 0.4 us of a call)
@functools.lru_cache(maxsize=1024)
def row_bytes(kind: int, cols: int) -> int:
    rb = lib().mi_row_bytes(kind, cols)
    if rb < 0:
        raise ValueError(f"{cols} values is not a whole number of type-{kind} blocks")
    return rb


class DeviceContext:
    """One device and one stream, like MAX's DeviceContext in the reference
    (one per process, tests/main.mojo:52-60).  Holds the workspace the
    library draws scratch from; it grows on demand and is reused.  Calls of one
    context and the graphs captured on it share that workspace and run one after
    the other: what is to overlap takes a context each, or workspaces of its own."""

    def __init__(self, device: int = 0, stream: torch.cuda.Stream | None = None):
        if not torch.cuda.is_available():
            raise RuntimeError("no GPU: the molla_amd kernels run only on a ROCm device")
        self.device = torch.device("cuda", device)
        self.index = self.device.index
        self.stream = stream if stream is not None else torch.cuda.current_stream(self.device)
        self._work = None
        self._captured = []  # workspaces that a captured graph replays on
        lib()  # fail now, not at the first launch, if the library is missing

    @property
    def handle(self) -> int:
        return self.stream.cuda_stream

    def workspace(self, nbytes: int) -> torch.Tensor:
        nbytes = max(int(nbytes), 256)
        if self._work is None or self._work.numel() < nbytes:
            # (of the stream that runs on it, so that one it replaces is reused in that order)
            with torch.cuda.stream(self.stream):
                self._work = torch.empty(nbytes + 256, dtype=torch.uint8, device=self.device)
        if torch.cuda.is_current_stream_capturing() and not any(w is self._work for w in self._captured):
            self._captured.append(self._work)
        return self._work

    def synchronize(self) -> None:
        check(lib().mi_sync(self.handle))


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _f32(t: torch.Tensor, name: str) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
        raise ValueError(f"{name} has to be a contiguous float32 device tensor")


def check_matvec_shapes(w: Tensor, x_elements: int, out_elements: int, tokens: int = 1) -> None:
    """gpu.mojo:2070 check_matvec_shapes, before anything is launched."""
    if w.place != WHERE_DEVICE:
        raise ValueError("the weight is not resident on the device")
    if x_elements < tokens * w.cols:
        raise ValueError(f"matvec wants an input of {tokens * w.cols} but got {x_elements}")
    if out_elements < tokens * w.rows:
        raise ValueError(f"matvec wants an output of {tokens * w.rows} but got {out_elements}")


def device_matvec_into(ctx: DeviceContext, w: Tensor, x: torch.Tensor, out: torch.Tensor, at: int = 0,
                       epi: int = EPI_NONE, aux: torch.Tensor | None = None) -> None:
    """out[at + r] = epilogue(dot(row r of w, x)); queued, not synchronized (gpu.mojo:2148)."""
    device_matmul_into(ctx, w, x, out, 1, at, epi, aux)


def device_matmul_into(ctx: DeviceContext, w: Tensor, x: torch.Tensor, out: torch.Tensor, tokens: int,
                       at: int = 0, epi: int = EPI_NONE, aux: torch.Tensor | None = None) -> None:
    """out[at + t*rows + r] = dot(row r of w, x[t]) for t < tokens (gpu.mojo:2945)."""
    if tokens <= 0:
        raise ValueError("a batched matmul needs at least one token")
    if at < 0:
        raise ValueError("a matvec cannot write at a negative offset")
    _f32(x, "x")
    _f32(out, "out")
    check_matvec_shapes(w, x.numel(), out.numel() - at, tokens)
    if aux is not None:
        _f32(aux, "aux")
    # with room for split-K partial sums when the chunk is a prefill one
    need = lib().mi_matmul_workspace(w.rows, w.cols, tokens)
    work = ctx.workspace(need)
    y = out.data_ptr() + 4 * at
    # aux defaults to the output when the epilogue does not read it (gpu.mojo:2217)
    a = aux.data_ptr() if (aux is not None and epi & (EPI_BIAS | EPI_GLU)) else y
    check(lib().mi_matvec(ctx.handle, w.kind, w.address, w.row_bytes(), w.rows, w.cols, x.data_ptr(), tokens,
                          y, epi, a, work.data_ptr(), work.numel()))


def device_matvec(ctx: DeviceContext, w: Tensor, x: np.ndarray, out: np.ndarray) -> None:
    """Host vectors either side: upload, launch, synchronize, download (gpu.mojo:3112)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    check_matvec_shapes(w, x.size, out.size)
    d_x = torch.from_numpy(x).to(ctx.device)
    d_o = torch.empty(w.rows, dtype=torch.float32, device=ctx.device)
    device_matvec_into(ctx, w, d_x, d_o)
    ctx.synchronize()
    out[:] = d_o.cpu().numpy()


def device_dequant(ctx: DeviceContext, w: Tensor, count: int | None = None) -> torch.Tensor:
    """The whole tensor (or its first `count` values) as float32, bit-exact to quant.mojo:412."""
    n = w.elements() if count is None else count
    out = torch.empty(n, dtype=torch.float32, device=ctx.device)
    check(lib().mi_dequant(ctx.handle, w.kind, w.address, n, out.data_ptr()))
    return out


def device_rms_norm(ctx: DeviceContext, out: torch.Tensor, x: torch.Tensor, gain: torch.Tensor, eps: float,
                    tokens: int = 1) -> None:
    """gpu_ops.mojo rms_norm: out = x * rsqrt(mean(x^2) + eps) * gain, per token row."""
    for t, n in ((out, "out"), (x, "x"), (gain, "gain")):
        _f32(t, n)
    n = gain.numel()
    if x.numel() != n * tokens or out.numel() != n * tokens:
        raise ValueError("rms_norm wants the input and the output the same size as the gain")
    check(lib().mi_rms_norm(ctx.handle, x.data_ptr(), gain.data_ptr(), n, tokens, eps, out.data_ptr(), None))


def rope_steps(dim: int, base: float) -> np.ndarray:
    """rope.mojo:230 step_table, computed on the host in float64."""
    out = np.zeros(dim // 2, dtype=np.float32)
    lib().mi_rope_steps(out.ctypes.data_as(ctypes.c_void_p), dim, base)
    return out


def device_rope(ctx: DeviceContext, x: torch.Tensor, heads: int, head_dim: int, dim: int, neox: bool,
                steps: torch.Tensor, pos: torch.Tensor, tokens: int = 1, row_stride: int | None = None) -> None:
    """Rotate heads in place at positions pos[t] (device int32)."""
    _f32(x, "x")
    stride = heads * head_dim if row_stride is None else row_stride
    check(lib().mi_rope(ctx.handle, x.data_ptr(), heads, head_dim, dim, int(neox), steps.data_ptr(),
                        pos.data_ptr(), tokens, stride))


CACHE_F16, CACHE_Q8 = 0, 1  # repack.mojo:174-181


@functools.lru_cache(maxsize=1024)
def cache_row(form: int, kv_width: int) -> int:
    """repack.mojo:221 cache_row: halves one cached position occupies."""
    row = lib().mi_cache_row(form, kv_width)
    if row < 0:
        raise ValueError(f"cache form {form} has no row of width {kv_width}")
    return row


def device_store_kv(ctx: DeviceContext, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                    v_cache: torch.Tensor, slot: int, form: int = CACHE_F16) -> None:
    """gpu_ops.mojo:1582 device_store_kv: f32 rows -> the cache at `slot`, f16
    or q8_0 (the caches are torch halves either way, cache_row per slot)."""
    kvw = k.numel()
    if v.numel() != kvw:
        raise ValueError("store_kv wants k and v the same width")
    row = cache_row(form, kvw)
    if k_cache.numel() < (slot + 1) * row or v_cache.numel() < (slot + 1) * row:
        raise ValueError(f"the cache has no room for slot {slot}")
    check(lib().mi_store_kv_form(ctx.handle, form, k.data_ptr(), v.data_ptr(), kvw, k_cache.data_ptr(),
                                 v_cache.data_ptr(), slot))


def device_attend(ctx: DeviceContext, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  heads: int, kv_heads: int, head_dim: int, scale: float, count: int,
                  out: torch.Tensor, form: int = CACHE_F16) -> None:
    """attention.mojo:144 attend over `count` cached positions (f16 or q8_0 cache)."""
    if count <= 0:
        raise ValueError("attention needs at least one key to look at")
    if k_cache.numel() < count * cache_row(form, kv_heads * head_dim):
        raise ValueError("attention wants more keys than the cache holds")
    need = lib().mi_attend_workspace(heads, head_dim, count)
    work = ctx.workspace(need)
    check(lib().mi_attend_form(ctx.handle, form, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), heads,
                               kv_heads, head_dim, scale, count, out.data_ptr(), work.data_ptr(), work.numel()))


def device_argmax(ctx: DeviceContext, x: torch.Tensor, n: int, tokens: int = 1) -> torch.Tensor:
    """kernel.mojo:571 argmax per token row, ties to the lower index."""
    out = torch.empty(tokens, dtype=torch.int32, device=ctx.device)
    check(lib().mi_argmax(ctx.handle, x.data_ptr(), n, tokens, out.data_ptr()))
    return out


def device_argmax_ws(ctx: DeviceContext, x: torch.Tensor, n: int, tokens: int = 1, next_ids=None,
                     next_pos=None) -> torch.Tensor:
    """device_argmax spread over 64 parts a row (mi_argmax_ws); next_ids /
    next_pos (device int32[tokens]) get the pick and pos + 1 when given."""
    L = lib()
    out = torch.empty(tokens, dtype=torch.int32, device=ctx.device)
    work = torch.empty(L.mi_argmax_workspace(n, tokens), dtype=torch.uint8, device=ctx.device)
    check(L.mi_argmax_ws(ctx.handle, x.data_ptr(), n, tokens, out.data_ptr(), work.data_ptr(), work.numel(),
                         None if next_ids is None else next_ids.data_ptr(),
                         None if next_pos is None else next_pos.data_ptr()))
    return out


def device_embed(ctx: DeviceContext, embedding: torch.Tensor, ids: torch.Tensor, out: torch.Tensor) -> None:
    """model.mojo:102 embed for an f32 table, one row per token id (device int32)."""
    vocab, width = embedding.shape
    check(lib().mi_embed(ctx.handle, embedding.data_ptr(), vocab, width, ids.data_ptr(), ids.numel(),
                         out.data_ptr()))


# ---- a step over trees of drafted tokens (no counterpart in the reference) ----
def _queue(ctx: DeviceContext, fn, *args) -> None:
    """A library call on the context's stream, with its device current."""
    if torch.cuda.current_device() == ctx.index:
        rc = fn(ctx.stream.cuda_stream, *args)
    else:
        with torch.cuda.device(ctx.index):
            rc = fn(ctx.stream.cuda_stream, *args)
    if rc:
        check(rc)


def _on(ctx: DeviceContext, t: torch.Tensor, name: str, dtype: torch.dtype, numel: int = 0) -> int:
    """The address of a contiguous tensor of the context's device, at least `numel` long."""
    if t.dtype is dtype and t.get_device() == ctx.index and t.is_contiguous() and (not numel or t.numel() >= numel):
        return t.data_ptr()
    if t.dtype is dtype and t.get_device() == ctx.index and t.is_contiguous():
        raise ValueError(f"{name} has {t.numel()} values where {numel} are needed")
    raise ValueError(f"{name} has to be a contiguous {dtype} tensor on {ctx.device}")


def _rows(ctx: DeviceContext, t: torch.Tensor, name: str, tokens: int, width: int) -> int:
    """The row stride of a float32 tensor of at least `tokens` rows of `width` values, each row contiguous."""
    if t.dtype is not torch.float32 or t.get_device() != ctx.index or t.dim() != 2:
        raise ValueError(f"{name} has to be float32 rows on {ctx.device}")
    rows, cols = t.shape
    stride, step = t.stride()
    if rows < tokens or cols < width or (step != 1 and cols > 1):
        raise ValueError(f"{name} has to be at least {tokens} x {width}, its rows contiguous")
    return stride if rows > 1 or stride > width else width


def device_page_plan(ctx: DeviceContext, page: int, lengths: torch.Tensor, news: torch.Tensor, table: torch.Tensor,
                     free_pages: torch.Tensor, free_count: torch.Tensor, free_left: torch.Tensor, starts: torch.Tensor,
                     seq: torch.Tensor | None, pos: torch.Tensor | None, cells: torch.Tensor,
                     kv_index: torch.Tensor | None = None) -> None:
    """Block tables and slot maps of a step (mi_page_plan): request b holds
    lengths[b] positions and gets news[b] more, in pages of `page` off the end of
    free_pages[:free_count].  Writes starts[batch + 1], the new pages into table
    [batch, pages], seq, pos and cells of every new token (as many rows as they
    have; seq and pos may be None), their entries of kv_index [batch, positions],
    and free_left = (pages left, pages wanted beyond them).  All int32.
    A request holds its table's first ceil(lengths[b] / page) pages and no others:
    after drafts were rejected the caller puts the pages behind the kept ones back,
    from free_pages[free_left[0]] on, ahead of the next plan."""
    i32 = torch.int32
    batch = lengths.numel()
    if table.dim() != 2 or table.shape[0] != batch or (kv_index is not None and (kv_index.dim() != 2 or
                                                                                 kv_index.shape[0] != batch)):
        raise ValueError(f"page_plan wants a table and a list a request ({batch})")
    tokens = cells.numel()
    _queue(ctx, lib().mi_page_plan, batch, page, _on(ctx, lengths, "lengths", i32), _on(ctx, news, "news", i32, batch),
           _on(ctx, table, "table", i32), table.shape[1], _on(ctx, free_pages, "free_pages", i32), free_pages.numel(),
           _on(ctx, free_count, "free_count", i32, 1), _on(ctx, free_left, "free_left", i32, 2),
           None if kv_index is None else _on(ctx, kv_index, "kv_index", i32),
           0 if kv_index is None else kv_index.shape[1], tokens, _on(ctx, starts, "starts", i32, batch + 1),
           None if seq is None else _on(ctx, seq, "seq", i32, tokens),
           None if pos is None else _on(ctx, pos, "pos", i32, tokens), _on(ctx, cells, "cells", i32))


def tree_words(max_nodes: int) -> int:
    """int32 words of a node's mask (mi_tree_words)."""
    words = lib().mi_tree_words(max_nodes)
    if words < 0:
        raise ValueError(f"a tree has 1 to 256 nodes, not {max_nodes}")
    return words


def device_tree_plan(ctx: DeviceContext, starts: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor,
                     max_nodes: int, pos: torch.Tensor | None, mask: torch.Tensor) -> None:
    """Ancestor masks and rotary positions of a step's trees (mi_tree_plan):
    parents[t] is the place in its own sequence of the node that token t follows,
    -1 for the committed tokens; mask [tokens, tree_words(max_nodes)] and pos
    [tokens] (or None), int32."""
    i32 = torch.int32
    batch, tokens = lengths.numel(), parents.numel()
    _queue(ctx, lib().mi_tree_plan, batch, _on(ctx, starts, "starts", i32, batch + 1),
           _on(ctx, lengths, "lengths", i32), _on(ctx, parents, "parents", i32), max_nodes, tokens,
           None if pos is None else _on(ctx, pos, "pos", i32, tokens),
           _on(ctx, mask, "mask", i32, tokens * tree_words(max_nodes)))


def device_qk_norm_rope(ctx: DeviceContext, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, heads: int,
                        kv_heads: int, head_dim: int, dim: int, neox: bool, steps: torch.Tensor, pos: torch.Tensor,
                        q_out: torch.Tensor, k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
                        cells: torch.Tensor | None = None, form: int = CACHE_F16, k_out: torch.Tensor | None = None,
                        q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-5,
                        factors: torch.Tensor | None = None, count: torch.Tensor | None = None) -> None:
    """Each head of q and k normed and rotated at pos[t], in one pass
    (mi_qk_norm_rope): q to q_out, k to k_out, and with v, the caches and cells
    (all four) k and v to the cache rows cells[t].  Rows are 2-D float32 views of
    any row stride; q_out may be q and k_out k.  count (device int32): rows from
    count on are left alone."""
    f32, i32 = torch.float32, torch.int32
    tokens = pos.numel()
    qw, kvw = heads * head_dim, kv_heads * head_dim

    def at(t, name, dtype, n=0):
        return None if t is None else _on(ctx, t, name, dtype, n)

    d = MiQk(heads, kv_heads, head_dim, dim, int(neox), form, tokens, eps, q.data_ptr(), k.data_ptr(),
             None if v is None else v.data_ptr(), _rows(ctx, q, "q", tokens, qw), _rows(ctx, k, "k", tokens, kvw),
             0 if v is None else _rows(ctx, v, "v", tokens, kvw), q_out.data_ptr(),
             None if k_out is None else k_out.data_ptr(), _rows(ctx, q_out, "q_out", tokens, qw),
             0 if k_out is None else _rows(ctx, k_out, "k_out", tokens, kvw), at(q_norm, "q_norm", f32, head_dim),
             at(k_norm, "k_norm", f32, head_dim), _on(ctx, steps, "steps", f32, dim // 2),
             at(factors, "factors", f32, dim // 2), _on(ctx, pos, "pos", i32), at(count, "count", i32, 1),
             at(k_cache, "k_cache", torch.float16), at(v_cache, "v_cache", torch.float16), at(cells, "cells", i32, tokens))
    _queue(ctx, lib().mi_qk_norm_rope, ctypes.byref(d))


def tree_cache(kv_index: torch.Tensor | None, batch: int, cache_stride: int, max_count: int, form: int,
               width: int) -> tuple:
    """(entries of a sequence's list of cells or 0, halves a cache holds at least) of a step over trees."""
    if kv_index is None:
        return 0, (batch - 1) * cache_stride + max_count * cache_row(form, width)
    if kv_index.dim() != 2 or kv_index.shape[0] < batch:
        raise ValueError(f"a step over trees wants a list of cells a sequence ({batch})")
    return kv_index.shape[1], 1


def device_attend_tree(ctx: DeviceContext, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int,
                       kv_heads: int, head_dim: int, scale: float, starts: torch.Tensor, lengths: torch.Tensor,
                       mask: torch.Tensor, max_nodes: int, max_count: int, out: torch.Tensor, cache_stride: int = 0,
                       kv_index: torch.Tensor | None = None, form: int = CACHE_F16,
                       work: torch.Tensor | None = None) -> None:
    """Attention of a step's trees over the caches (mi_attend_tree): q [tokens,
    heads * head_dim] (rows of any stride), out the same contiguous.  Sequence b's
    slots are rows of its own cache, cache_stride halves after the one before, or
    the cells kv_index[b]; lengths[b] of them are committed, its nodes behind."""
    i32, f16 = torch.int32, torch.float16
    batch, tokens = lengths.numel(), q.shape[0]
    qw = heads * head_dim
    q_stride = _rows(ctx, q, "q", tokens, qw)
    stride, least = tree_cache(kv_index, batch, cache_stride, max_count, form, kv_heads * head_dim)
    tree = MiTree(batch, tokens, max_nodes, max_count, _on(ctx, starts, "starts", i32, batch + 1),
                  _on(ctx, lengths, "lengths", i32), _on(ctx, mask, "mask", i32, tokens * tree_words(max_nodes)))
    L = lib()
    t = ctypes.byref(tree)
    if work is None:
        work = ctx.workspace(L.mi_attend_tree_workspace(heads, kv_heads, head_dim, form, t))
    else:
        _on(ctx, work, "work", torch.uint8)
    _queue(ctx, L.mi_attend_tree, form, q.data_ptr(), q_stride, _on(ctx, k_cache, "k_cache", f16, least),
           _on(ctx, v_cache, "v_cache", f16, least), cache_stride,
           None if kv_index is None else _on(ctx, kv_index, "kv_index", i32), stride, heads, kv_heads, head_dim, scale,
           t, _on(ctx, out, "out", torch.float32, tokens * qw), work.data_ptr(), work.numel())


def device_attend_window(ctx: DeviceContext, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int,
                         kv_heads: int, head_dim: int, scale: float, window: int, first: int, pos: torch.Tensor,
                         max_count: int, out: torch.Tensor, cache_stride: int = 0, kv_index: torch.Tensor | None = None,
                         form: int = CACHE_F16, work: torch.Tensor | None = None) -> None:
    """Attention over the last `window` positions and the first few (mi_attend_window):
    the token of row t of q [tokens, heads * head_dim] (rows of any stride) is at
    position pos[t] (int32) of its sequence and sees the positions up to its own that
    are above pos[t] - window or below `first`.  Its sequence's cache lies cache_stride
    halves after the one before, or kv_index [tokens, positions] lists its pool cells;
    a cache_stride of 0, or one list [positions], makes the rows one sequence's chunk.
    max_count bounds the positions.  out is as q, contiguous."""
    f16, i32 = torch.float16, torch.int32
    tokens, qw = pos.numel(), heads * head_dim
    row = cache_row(form, kv_heads * head_dim)
    stride = 0
    if kv_index is not None:
        if kv_index.dim() not in (1, 2) or (kv_index.dim() == 2 and kv_index.shape[0] != tokens):
            raise ValueError(f"attend_window wants one list of cells, or one for each of {tokens} tokens")
        if kv_index.shape[-1] < max_count:
            raise ValueError(f"attend_window: a list of {kv_index.shape[-1]} cells for {max_count} positions")
        stride = kv_index.shape[1] if kv_index.dim() == 2 else 0
        least = 1
    else:
        least = (tokens - 1) * cache_stride + max_count * row
    L = lib()
    if work is None:
        work = ctx.workspace(L.mi_attend_window_workspace(heads, kv_heads, head_dim, form, window, first, max_count, tokens,
                                                          int((cache_stride if kv_index is None else stride) == 0)))
    _queue(ctx, L.mi_attend_window, form, q.data_ptr(), _rows(ctx, q, "q", tokens, qw),
           _on(ctx, k_cache, "k_cache", f16, least), _on(ctx, v_cache, "v_cache", f16, least), cache_stride,
           None if kv_index is None else _on(ctx, kv_index, "kv_index", i32), stride, heads, kv_heads, head_dim, scale,
           window, first, _on(ctx, pos, "pos", i32), max_count, tokens, _on(ctx, out, "out", torch.float32, tokens * qw),
           _on(ctx, work, "work", torch.uint8), work.numel())


# ---- sparse experts (no counterpart in the reference) ----
ROUTER_SIGMOID, ROUTER_NORM = 1, 2


def device_router(ctx: DeviceContext, x: torch.Tensor, router: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                  bias: torch.Tensor | None = None, sigmoid: bool = False, norm: bool = True, scale: float = 1.0,
                  work: torch.Tensor | None = None) -> None:
    """Which experts each row of x [tokens, width] takes (mi_router): router
    [experts, width] f32; writes ids [tokens, used] (int32) and weights the same
    (f32).  Scores are the softmax over the experts, or sigmoid each; bias [experts]
    is added for the choice alone; norm: a token's weights sum to scale."""
    f32 = torch.float32
    if x.dim() != 2 or router.dim() != 2 or ids.dim() != 2 or x.shape[1] != router.shape[1]:
        raise ValueError("router wants x [tokens, width], router [experts, width] and ids [tokens, used]")
    (tokens, width), experts, used = x.shape, router.shape[0], ids.shape[1]
    if ids.shape[0] != tokens or weights.shape != ids.shape:
        raise ValueError(f"router wants ids and weights for {tokens} tokens, alike")
    L = lib()
    work = ctx.workspace(L.mi_router_workspace(experts, tokens)) if work is None else work
    _queue(ctx, L.mi_router, _on(ctx, x, "x", f32), _on(ctx, router, "router", f32),
           None if bias is None else _on(ctx, bias, "bias", f32, experts), width, experts, used, tokens,
           (ROUTER_SIGMOID if sigmoid else 0) | (ROUTER_NORM if norm else 0), scale, _on(ctx, ids, "ids", torch.int32),
           _on(ctx, weights, "weights", f32), _on(ctx, work, "work", torch.uint8), work.numel())


def _stacked(w: Tensor, experts: int, name: str) -> int:
    """Rows of one expert of a stacked tensor."""
    if experts < 1 or w.rows % experts:
        raise ValueError(f"{name} has {w.rows} rows, which are no {experts} experts")
    return w.rows // experts


def device_experts_matmul(ctx: DeviceContext, w: Tensor, experts: int, x: torch.Tensor, ids: torch.Tensor,
                          out: torch.Tensor, work: torch.Tensor | None = None) -> None:
    """Matrix products grouped by expert (mi_experts_matmul): w stacks `experts`
    matrices; out [pairs, rows] row p is expert ids[p]'s matrix against x [pairs /
    share, cols] row p / share.  A row whose id is no expert keeps what it held."""
    f32 = torch.float32
    rows, pairs = _stacked(w, experts, "w"), ids.numel()
    if x.dim() != 2 or x.shape[1] != w.cols or not x.shape[0] or pairs % x.shape[0]:
        raise ValueError(f"experts_matmul wants x of whole rows of {w.cols} for {pairs} ids")
    share = pairs // x.shape[0]
    L = lib()
    work = ctx.workspace(L.mi_experts_matmul_workspace(experts, w.cols, share, pairs)) if work is None else work
    _queue(ctx, L.mi_experts_matmul, w.kind, w.address, w.row_bytes(), experts, rows, w.cols, _on(ctx, x, "x", f32), share,
           _on(ctx, ids, "ids", torch.int32), pairs, _on(ctx, out, "out", f32, pairs * rows),
           _on(ctx, work, "work", torch.uint8), work.numel())


def device_experts_mlp(ctx: DeviceContext, gate: Tensor, up: Tensor, down: Tensor, experts: int, x: torch.Tensor,
                       ids: torch.Tensor, weights: torch.Tensor, out: torch.Tensor, act: int = 0, add: bool = False,
                       work: torch.Tensor | None = None) -> None:
    """The experts' gated MLP and its weighted sum (mi_experts_mlp): x and out
    [tokens, width], ids and weights [tokens, used]; gate, up and down stack
    `experts` matrices.  act: 0 silu, ACT_BIT gelu; add: onto what out holds."""
    f32 = torch.float32
    if x.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0] or weights.shape != ids.shape:
        raise ValueError("experts_mlp wants x [tokens, width] with ids and weights [tokens, used]")
    (tokens, width), used = x.shape, ids.shape[1]
    d = MiExperts(experts, width, _stacked(gate, experts, "gate"), act, gate.weight(), up.weight(), down.weight())
    L, p = lib(), ctypes.byref(d)
    work = ctx.workspace(L.mi_experts_workspace(p, tokens, used)) if work is None else work
    _queue(ctx, L.mi_experts_mlp, p, _on(ctx, x, "x", f32), tokens, used, _on(ctx, ids, "ids", torch.int32),
           _on(ctx, weights, "weights", f32), _on(ctx, out, "out", f32, tokens * width), EPI_ADD if add else EPI_NONE,
           _on(ctx, work, "work", torch.uint8), work.numel())


__all__ = [n for n in dir() if not n.startswith("_")] + ["MiError"]
