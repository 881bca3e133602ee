"""The 4-bit KV cache (aljabr_blackwell_kv4_*): quantise rows as they are
written, read them back, and attend over them.

A cache is a pool of pages; a sequence owns pages through a block table, or
one page of max_ctx positions each (no table).  The serving loop of one layer:

    cache = Kv4Cache(pages, page_size, kv_heads, head_dim)
    cache.append(k, v, slots)                      # new rows -> 4 bits
    out = cache.attend(q, seq_lens, block_table)   # q: [batch, q_len, q_heads, head_dim]

Speculative decoding drafts a tree of tokens a sequence, whose nodes take the
positions behind it (parents: int32, -1 a root, -2 an absent node).  One step:

    q = cache.append_rotated(q, k, v, slots, positions, rope)    # each layer
    out = cache.attend_tree(q, seq_lens, parents, block_table)
    ...                                                          # logits, process_logits: picked
    path, count, token, lens = accept_tree(caches, seq_lens, parents, drafted, picked, block_table)

Tensors are torch CUDA tensors on the cache's device; every call is ordered on
torch's current stream of that device (or `stream`, a raw cudaStream_t: what
the call is given must be ready there and live until it has run), and may be
captured with torch.cuda.graph.  The layout and the arithmetic are described
in include/aljabr_blackwell.h.
"""
from __future__ import annotations

import ctypes
import functools
import os
import threading
import warnings

import torch

from . import native

_DTYPES = {torch.float32: native.KV_F32, torch.bfloat16: native.KV_BF16}
_LEGACY_STREAM = 1      # cudaStreamLegacy: the C-ABI reads 0 as "the library's own stream"
_THREAD_STREAM = 2      # cudaStreamPerThread: another stream in each thread


# torch.cuda.current_stream(device).cuda_stream without building the Stream object (2.6 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def current_stream(index: int) -> int:
    return _raw_stream(index) or _LEGACY_STREAM


class selected:
    """Device `index` selected in the library, which launches on the calling thread's device, and in CUDA; on leaving,
    both choices are the caller's again."""

    def __init__(self, index: int):
        self.index, self.library = index, ctypes.c_int(-1)

    def __enter__(self):
        self.cuda = torch.cuda.current_device()
        native.call("aljabr_blackwell_device_swap", self.index, ctypes.byref(self.library))

    def __exit__(self, *exc):
        native.call("aljabr_blackwell_device_swap", self.library.value, ctypes.byref(ctypes.c_int(-1)))
        torch.cuda.set_device(self.cuda)


def selecting(call, index_of):
    """`call` on the device that index_of finds in its arguments; where there is one device, `call` itself."""
    if torch.cuda.device_count() <= 1:
        return call

    @functools.wraps(call)
    def on_device(*args, **kwargs):
        index = index_of(*args, **kwargs)
        if index < 0:
            return call(*args, **kwargs)      # not a CUDA tensor: refused there
        with selected(index):
            return call(*args, **kwargs)
    return on_device


def stream_key(stream: int):
    """What tells streams apart whose calls do not follow one another."""
    return stream if stream != _THREAD_STREAM else (stream, threading.get_ident())


def capture_id(stream: int) -> int:
    """Id of the graph capture that `stream` takes part in; 0 where it is in none."""
    got = ctypes.c_ulonglong(0)
    native.call("aljabr_blackwell_stream_capture_id", stream, ctypes.byref(got))
    return got.value


def torch_stream(stream: int, device):
    """The handle as torch's object.  Torch reads an odd number, as the legacy stream's is, as one of its own streams."""
    return torch.cuda.default_stream(device) if stream == _LEGACY_STREAM else torch.cuda.ExternalStream(stream, device)


def new_output(shape, dtype, device, index: int, stream: int) -> torch.Tensor:
    """A tensor that a call on `stream` writes and that the caller reads on torch's current stream: of the allocator's
    pool of the first, so that no work pending on the second still uses its memory, and not given out again before
    the second is done with it."""
    if stream == current_stream(index):
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(torch_stream(stream, device)):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(torch.cuda.current_stream(device))
    return t


_tree_work = {}     # (device, stream_key) -> workspace of attend_tree, of all caches: calls on one stream follow one another
_making = threading.Lock()      # workspaces are made once: a thread's launch may still be coming with the address of the first
_kinds = {}         # shapes of caches
_captured = {}      # (device, stream_key) -> capture id, its workspaces
_kept = []          # workspaces of captures on streams given by handle


def dtype_id(t: torch.Tensor, what: str) -> int:
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise native.UnsupportedOperation(native.ALJ_ERR_UNSUPPORTED, f"{what} is {t.dtype}: float32 or bfloat16")
    return d


def bad(message: str) -> native.ProviderError:
    return native.ProviderError(native.ALJ_ERR_BAD_ARG, message)


def _load_calls():
    """tensor_calls.so, where it was built and with this torch.  It takes tensors to the library in less host time; without
    it every call goes through ctypes, to the same kernels."""
    try:
        from . import tensor_calls
        made = getattr(tensor_calls, "torch", "of another version")
        if made == torch.__version__:
            return tensor_calls
        why = f"it was built with torch {made}"
    except ImportError as e:
        if not os.path.exists(os.path.join(os.path.dirname(__file__), "tensor_calls.so")):
            return None
        why = str(e)
    warnings.warn(f"tensor_calls.so is not used ({why}): calls take more host time until `python -m aljabr_b200.build`",
                  RuntimeWarning, stacklevel=3)
    return None


tensor_calls = _load_calls()


class Kv4Cache:
    """`pages` pages of `page_size` positions of `kv_heads` heads in 4 bits.

    `data`: uint8 storage to use (for example another process's or layer's
    share of one allocation); a zeroed buffer is allocated without it.
    """

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda", data=None):
        size = native.lib().aljabr_blackwell_kv4_cache_size(pages, page_size, kv_heads, head_dim)
        if size < 0:
            native.check(int(size))
        if data is None:
            data = torch.zeros(size, dtype=torch.uint8, device=device)
        if data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() < size or data.device.type != "cuda":
            raise bad(f"cache data must be {size} contiguous uint8 on a CUDA device")
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self.data, self.device, self.bytes = data, data.device, size
        self._index = data.get_device()
        with selected(self._index):
            native.call("aljabr_blackwell_init", self._index)      # refuses other GPUs than the library's
        lib = native.lib()
        self._append, self._read = lib.aljabr_blackwell_kv4_append_dev, lib.aljabr_blackwell_kv4_read_dev
        self._attend, self._work_size = lib.aljabr_blackwell_kv4_attention_dev, lib.aljabr_blackwell_kv4_attention_workspace_size
        self._row = kv_heads * head_dim
        self._address = data.data_ptr()
        # one object for all caches of a shape on a device
        self._kind = _kinds.setdefault(k := (pages, page_size, kv_heads, head_dim, self._index), k)
        self._shape = (data.data_ptr(), pages, page_size, kv_heads, head_dim)
        self._buffers = {}   # stream_key -> workspace: calls on one stream never overlap
        self._work = {}      # (stream_key, q_len, q_heads) -> its address and size

    # -- checks ----------------------------------------------------------------
    def _rows(self, t: torch.Tensor, tokens: int, what: str) -> int:
        """Elements between the rows of t: [tokens, kv_heads, head_dim] or [tokens, kv_heads * head_dim]."""
        shape, st = t.shape, t.stride()
        if len(shape) == 3:
            ok = shape == (tokens, self.kv_heads, self.head_dim) and (st[1] == self.head_dim or self.kv_heads == 1)
        else:
            ok = shape == (tokens, self._row)
        if not ok or st[-1] != 1 or t.get_device() != self._index:
            raise bad(f"{what} must be [{tokens}, {self.kv_heads}, {self.head_dim}] on {self.device} with contiguous rows, "
                      f"not {tuple(shape)} with strides {st} on {t.device}")
        return st[0] if tokens > 1 else self._row

    def _ints(self, t: torch.Tensor, n: int, what: str) -> int:
        if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != n or t.get_device() != self._index or not t.is_contiguous():
            raise bad(f"{what} must be contiguous int32 [{n}] on {self.device}")
        return t.data_ptr()

    def _dense(self, t, tokens: int, dtype, what: str):
        if t is None:
            return None
        if t.dtype is not dtype or t.numel() != tokens * self._row or t.get_device() != self._index or not t.is_contiguous():
            raise bad(f"{what} must be contiguous {dtype} [{tokens}, {self.kv_heads}, {self.head_dim}] on {self.device}")
        return t.data_ptr()

    # -- rows ------------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_back=None, v_back=None, stream=None):
        """Quantise the rows k, v into slots[i] = page * page_size + position (-1: skip the row).

        k_back / v_back (both or neither) receive the values the cache now holds."""
        n, dtype = slots.numel(), k.dtype
        kind = _DTYPES.get(dtype)
        if kind is None:
            dtype_id(k, "k")
        if v.dtype is not dtype:
            raise bad(f"k is {dtype}, v is {v.dtype}")
        ks, vs = self._rows(k, n, "k"), self._rows(v, n, "v")
        kb = None if k_back is None else self._dense(k_back, n, dtype, "k_back")
        vb = None if v_back is None else self._dense(v_back, n, dtype, "v_back")
        rc = self._append(*self._shape, k.data_ptr(), v.data_ptr(), kind, ks, vs, self._ints(slots, n, "slots"), n, kb, vb,
                          stream or current_stream(self._index))
        if rc:
            native.check(rc)

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                       rope: torch.Tensor, interleaved: bool = False, q_out=None, k_back=None, v_back=None,
                       stream=None) -> torch.Tensor:
        """append() with the rotation of q and k by their positions on the way; returns the rotated q.

        q: [tokens, q_heads, head_dim] with contiguous rows, of k's type.  positions: int32 [tokens], below zero where a
        token is absent (its q is zero, nothing is stored).  rope: float32 [positions, n, 2] of (cos, sin), contiguous;
        a head's first 2 n dims turn, dims i and i + n a pair, or with `interleaved` 2 i and 2 i + 1.  q_out: of q's
        shape and type, its rows may be strided; q itself will do.  k_back, v_back: as for append(); k and v themselves will do.
        Outputs may lie between the rows of other arguments, but overlap none."""
        got = tensor_calls.rotate_append(*self._shape, self._index, q, k, v, slots, positions, rope, interleaved, q_out, k_back, v_back,
                                         stream) if tensor_calls else NotImplemented
        if got is not NotImplemented:
            return native.check(got) if type(got) is int else got
        n, dtype = slots.numel(), k.dtype
        kind = _DTYPES.get(dtype)
        if kind is None:
            dtype_id(k, "k")
        if v.dtype is not dtype or q.dtype is not dtype:
            raise bad(f"k is {dtype}, v is {v.dtype}, q is {q.dtype}")
        ks, vs = self._rows(k, n, "k"), self._rows(v, n, "v")
        heads = q.shape[1] if q.dim() == 3 else 0
        qs = self._q_rows(q, n, heads, "q")
        if rope.dtype is not torch.float32 or rope.dim() != 3 or rope.shape[2] != 2 or rope.get_device() != self._index or \
                not rope.is_contiguous():
            raise bad(f"rope must be contiguous float32 [positions, pairs, 2] on {self.device}")
        if max(n, rope.shape[0]) > 0x7FFFFFFF:       # ctypes would take their low 32 bits
            raise bad(f"{n} tokens, {rope.shape[0]} positions of rope: each at most 2^31 - 1")
        kb = None if k_back is None else self._dense(k_back, n, dtype, "k_back")
        vb = None if v_back is None else self._dense(v_back, n, dtype, "v_back")
        stream = stream or current_stream(self._index)
        if q_out is None:
            q_out = new_output(q.shape, dtype, self.device, self._index, stream)
        elif q_out.dtype is not dtype:
            raise bad(f"q is {dtype}, q_out is {q_out.dtype}")
        rc = native.lib().aljabr_blackwell_kv4_rotate_append_dev(
            *self._shape, q_out.data_ptr(), self._q_rows(q_out, n, heads, "q_out"), q.data_ptr(), k.data_ptr(), v.data_ptr(), kind,
            qs, ks, vs, heads, self._ints(slots, n, "slots"), self._ints(positions, n, "positions"), rope.data_ptr(), rope.shape[0],
            2 * rope.shape[1], bool(interleaved), n, kb, vb, stream)
        if rc:
            native.check(rc)
        return q_out

    def _q_rows(self, t: torch.Tensor, tokens: int, heads: int, what: str) -> int:
        shape, st, D = t.shape, t.stride(), self.head_dim
        if shape != (tokens, heads, D) or st[2] != 1 or (heads > 1 and st[1] != D) or t.get_device() != self._index:
            raise bad(f"{what} must be [{tokens}, q_heads, {D}] on {self.device} with contiguous rows, "
                      f"not {tuple(shape)} with strides {st} on {t.device}")
        return st[0] if tokens > 1 else heads * D

    def read(self, slots: torch.Tensor, dtype=torch.float32, k_out=None, v_out=None, stream=None):
        """Rows of the given slots as (k, v), [n, kv_heads, head_dim] each; zeros where a slot is -1."""
        n = slots.numel()
        stream = stream or current_stream(self._index)
        if k_out is None and v_out is None:
            k_out, v_out = (new_output((n, self.kv_heads, self.head_dim), dtype, self.device, self._index, stream) for _ in range(2))
        some = k_out if k_out is not None else v_out
        rc = self._read(self._dense(k_out, n, some.dtype, "k_out"), self._dense(v_out, n, some.dtype, "v_out"),
                        dtype_id(some, "k_out"), *self._shape, self._ints(slots, n, "slots"), n, stream)
        if rc:
            native.check(rc)
        return k_out, v_out

    # -- attention -------------------------------------------------------------
    def _workspace(self, q_len: int, q_heads: int, stream: int):
        """(address, bytes) of this stream's workspace: made once, as large as any accepted call needs (a few MB), and
        kept as long as the cache, since kernels under way may hold its address."""
        key = stream_key(stream)
        have = self._buffers.get(key)
        if have is None:
            with _making:
                have = self._buffers.get(key)
                if have is None:
                    have = self._buffers[key] = self._make_workspace(q_len, q_heads, stream)
        got = self._work[key, q_len, q_heads] = (have.data_ptr(), have.numel())
        return got

    def _make_workspace(self, q_len: int, q_heads: int, stream: int) -> torch.Tensor:
        need = self._work_size(q_len, q_heads, self.kv_heads, self.head_dim)   # the call's own, for its refusals
        if need < 0:
            native.check(int(need))
        return self._zeros(self._work_size(native.KV4_MAX_ROWS, self.kv_heads, self.kv_heads, self.head_dim), stream)

    def _tree_workspace(self, stream: int):
        """(address, bytes) of this stream's workspace for trees: as large as any call of any cache needs (39 MB), and kept for
        good, since kernels under way may hold its address."""
        key = self._index, stream_key(stream)
        have = _tree_work.get(key)
        if have is None:
            size, group = native.lib().aljabr_blackwell_kv4_tree_attention_workspace_size, native.KV4_MAX_ROWS // native.KV4_MAX_NODES
            most = max(size(native.KV4_MAX_NODES, group, 1, D) for D in (64, 128, 256))
            with _making:
                have = _tree_work.get(key)
                if have is None:
                    have = _tree_work[key] = self._zeros(int(most), stream)
        return have.data_ptr(), have.numel()

    def _zeros(self, size: int, stream: int) -> torch.Tensor:
        """Made and zeroed on the stream whose kernels will use it."""
        if stream == current_stream(self._index):
            return torch.zeros(size, dtype=torch.uint8, device=self.device)
        with torch.cuda.stream(torch_stream(stream, self.device)):
            return torch.zeros(size, dtype=torch.uint8, device=self.device)

    def _captured_workspace(self, capture: int, q_len: int, q_heads: int, stream: int, tree: bool = False):
        """(address, bytes) for calls recorded into a graph.  Its zeroing is a node of that graph, which may run on any
        stream: so it belongs to this capture's calls on this stream (of all caches: they follow one another) and to
        nothing else.  torch's graph keeps the memory: here it is held until the stream's next capture, and for good
        where the stream was given by its handle, since other means of capture keep nothing."""
        key = self._index, stream_key(stream)
        owner, have = _captured.get(key, (0, []))
        if owner != capture:
            _captured[key] = capture, (have := [])
        size = native.lib().aljabr_blackwell_kv4_tree_attention_workspace_size if tree else self._work_size
        need = size(q_len, q_heads, self.kv_heads, self.head_dim)
        if need < 0:
            native.check(int(need))
        if not have or have[-1].numel() < need:
            have.append(self._zeros(int(need), stream) if tree else self._make_workspace(q_len, q_heads, stream))
            if stream != current_stream(self._index):
                _kept.append(have[-1])
        return have[-1].data_ptr(), have[-1].numel()

    def attend(self, q: torch.Tensor, seq_lens: torch.Tensor, block_table=None, window: int = 0, scale=None,
               soft_cap: float = 0.0, out=None, stream=None) -> torch.Tensor:
        """Attention of q [batch, q_len, q_heads, head_dim], whose rows are the last q_len of seq_lens[b] positions.

        block_table: int32 [batch, pages a sequence], or None where sequence b is page b.  scale: 1 / sqrt(head_dim)
        by default.  Returns out, contiguous, of q's type."""
        return self._attention(q, seq_lens, None, block_table, window, scale, soft_cap, out, stream)

    def attend_tree(self, q: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor, block_table=None, window: int = 0,
                    scale=None, soft_cap: float = 0.0, out=None, stream=None) -> torch.Tensor:
        """Attention of the nodes of drafted trees, the last `nodes` of seq_lens[b] positions: q [batch, nodes, q_heads,
        head_dim].  A node sees the positions before the tree, its ancestors and itself; zeros where it is absent.

        parents: int32 [batch, nodes], or [nodes] for one tree of all sequences; -1 a root, -2 absent, else an earlier
        node.  window counts a node by its depth.  The rest as attend()."""
        nodes = q.shape[1] if q.dim() == 4 else -1
        if parents.dtype is not torch.int32 or parents.shape not in ((nodes,), (q.shape[0], nodes)) or \
                parents.get_device() != self._index or not parents.is_contiguous():
            raise bad(f"parents must be contiguous int32 [{nodes}] or [{q.shape[0]}, {nodes}] on {self.device}")
        return self._attention(q, seq_lens, parents, block_table, window, scale, soft_cap, out, stream)

    def _attention(self, q, seq_lens, parents, block_table, window, scale, soft_cap, out, stream):
        shape, st = q.shape, q.stride()
        if len(shape) != 4 or shape[3] != self.head_dim or q.get_device() != self._index:
            raise bad(f"q must be [batch, q_len, q_heads, {self.head_dim}] on {self.device}, not {tuple(shape)} on {q.device}")
        batch, q_len, q_heads, D = shape
        q_stride = st[1] if q_len > 1 else st[0] if batch > 1 else q_heads * D
        if st[3] != 1 or (q_heads > 1 and st[2] != D) or (q_len > 1 and batch > 1 and st[0] != q_len * st[1]):
            raise bad(f"q: the heads of a token must be contiguous and the tokens evenly spaced (strides {st})")
        kind = dtype_id(q, "q")
        current = current_stream(self._index)
        stream = stream or current
        if out is None:
            out = new_output((batch, q_len, q_heads, D), q.dtype, self.device, self._index, stream)
        elif out.shape != shape or out.dtype is not q.dtype or out.get_device() != self._index or not out.is_contiguous():
            raise bad(f"out must be contiguous {q.dtype} {tuple(shape)} on {self.device}")
        table, width = None, 0
        if block_table is not None:
            width = block_table.shape[-1]
            # an empty table has no address, which would read as no table
            if block_table.dtype is not torch.int32 or block_table.shape != (batch, width) or (width == 0 and batch > 0) or \
                    block_table.get_device() != self._index or not block_table.is_contiguous():
                raise bad(f"block_table must be contiguous int32 [{batch}, 1 or more pages a sequence] on {self.device}")
            table = block_table.data_ptr()
        if window:       # ctypes would take its low 32 bits
            window = max(-1, min(window, 0x7FFFFFFF))
        capture = 0      # the legacy stream is never captured: no question asked there (0.8 us)
        if stream != _LEGACY_STREAM and (stream != current or torch.cuda.is_current_stream_capturing()):
            capture = capture_id(stream)
        if capture:
            work, size = self._captured_workspace(capture, q_len, q_heads, stream, parents is not None)
        elif parents is not None:
            work, size = self._tree_workspace(stream)
        else:
            have = self._work.get((stream_key(stream), q_len, q_heads))
            work, size = have if have is not None else self._workspace(q_len, q_heads, stream)
        scale = D ** -0.5 if scale is None else scale
        lens = self._ints(seq_lens, batch, "seq_lens")
        if parents is None:
            rc = self._attend(out.data_ptr(), q.data_ptr(), kind, q_stride, *self._shape, table, width, lens, batch, q_len,
                              q_heads, window, scale, soft_cap, work, size, stream)
        else:
            rc = native.lib().aljabr_blackwell_kv4_tree_attention_dev(
                out.data_ptr(), q.data_ptr(), kind, q_stride, *self._shape, table, width, lens, batch, parents.data_ptr(),
                q_len if parents.dim() == 2 else 0, q_len, q_heads, window, scale, soft_cap, work, size, stream)
        if rc:
            native.check(rc)
        return out


def accept_tree(caches, seq_lens: torch.Tensor, parents: torch.Tensor, drafted: torch.Tensor, picked: torch.Tensor,
                block_table=None, out=None, stream=None):
    """Keeps the drafted path that agrees with the model, in every cache of a list (a model's layers, of one shape).

    From node 0, the token emitted last, on to the first child whose drafted token is the one picked after its parent.
    drafted, picked: int32 [batch, nodes]; seq_lens, parents, block_table as for attend_tree.  The path's rows move to
    the first positions of the tree.  Returns int32 (path [batch, nodes], -1 behind its end; count [batch]; token
    [batch], picked after the path's last node; lens [batch], the sequence with its path), written to `out` where
    that is a result of an earlier call.  A sequence without a tree: count 0, token -1, its length."""
    caches = [caches] if isinstance(caches, Kv4Cache) else list(caches)
    if not caches:
        raise bad("no caches")
    first = caches[0]
    kind = first._kind
    addresses = [c._address for c in caches if c._kind is kind]
    if len(addresses) != len(caches):
        raise bad("the caches of one call must have the same shape and device")
    got = tensor_calls.accept_tree(addresses, *kind, seq_lens, parents, drafted, picked, block_table, out, stream) \
        if tensor_calls else NotImplemented
    if got is not NotImplemented:
        return native.check(got) if type(got) is int else got
    if drafted.dim() != 2:
        raise bad("drafted must be int32 [batch, nodes]")
    batch, nodes = drafted.shape
    ints = (lambda t, shapes, what: _int_tensor(t, shapes, what, first))
    stream = stream or current_stream(first._index)
    if out is None:
        out = tuple(new_output(s, torch.int32, first.device, first._index, stream) for s in ((batch, nodes),) + ((batch,),) * 3)
    table, width = None, 0
    if block_table is not None:
        width = block_table.shape[-1]
        table = ints(block_table, ((batch, max(width, 1)),), "block_table")
    path, count, token, lens = (ints(t, (s,), w) for t, s, w in zip(out, ((batch, nodes),) + ((batch,),) * 3,
                                                                    ("path", "count", "token", "lens")))
    rc = native.lib().aljabr_blackwell_kv4_accept_tree_dev(
        path, count, token, lens, (ctypes.c_void_p * len(caches))(*addresses), len(caches), *first._shape[1:], table, width,
        ints(seq_lens, ((batch,),), "seq_lens"), batch, ints(parents, ((nodes,), (batch, nodes)), "parents"),
        nodes if parents.dim() == 2 else 0, nodes, ints(drafted, ((batch, nodes),), "drafted"),
        ints(picked, ((batch, nodes),), "picked"), stream)
    if rc:
        native.check(rc)
    return out


def _int_tensor(t: torch.Tensor, shapes, what: str, cache: Kv4Cache) -> int:
    if t.dtype is not torch.int32 or t.shape not in shapes or t.get_device() != cache._index or not t.is_contiguous():
        raise bad(f"{what} must be contiguous int32 {' or '.join(str(list(s)) for s in shapes)} on {cache.device}, "
                  f"not {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _index_of(caches, *_, **__):
    caches = [caches] if isinstance(caches, Kv4Cache) else list(caches)
    return caches[0]._index if caches else -1


accept_tree = selecting(accept_tree, _index_of)
for _name in ("append", "append_rotated", "read", "attend", "attend_tree"):
    setattr(Kv4Cache, _name, selecting(getattr(Kv4Cache, _name), lambda cache, *_, **__: cache._index))
