"""Host side of the 8-bit paged KV cache.

``Kv8Cache`` holds one attention layer's whole context in 8 bits (float8 e4m3
or int8), with a scale for each block of 64 tokens and head, in pages that a
table assigns to the sequences: half the bytes of a 16-bit cache for decode to
read.  The up to 63 tokens behind a sequence's last complete block stay in
16 bits, so what the cache holds depends on the tokens alone.  The layout and
semantics are documented with ``nsa_kv8_cache`` in include/nsa_b200.h; the
reference has no counterpart.

Beside the other caches: ``KiviCache`` keeps a window at 2 bits, ``RingCache``
a window at 16 bits, ``Kv8Cache`` every token (and attends to all of them or
to sink + window).  It takes float16 or bfloat16, head_dim 64 or 128, any
number of query heads per KV head, ragged batches and several query tokens.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib
from .constants import D_HEAD, SINK_SIZE

BLOCK = 64    # tokens of a page and of a scale
RING = 128    # 16-bit slots of a sequence: the incomplete block and the one before it
MAX_QUERY = 64  # query tokens of one attend

_CODES = {"e4m3": (0, torch.float8_e4m3fn), "int8": (1, torch.int8)}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# Scratch of attention.  Eager calls share one (workspace, tickets) pair per
# (device, stream).  A call captured into a graph takes its workspace from the
# graph's own pool and a ticket row for itself, so that graphs replayed side by
# side do not share them.  A row may be its graph's for as long as the process
# lives, so it is not handed out again: after _GRAPH_ROWS calls tickets come from
# the graph's pool, where the graph zeroes them before each (one more node).
_GRAPH_ROWS = 4096
_scratch_lock = threading.Lock()
_eager: dict = {}
_graph: dict = {}  # device index -> [rows, rows handed out]


def _graph_rows(device):
    """Ticket rows for captured calls, made before any capture (when a cache is)."""
    with _scratch_lock:
        if device.index not in _graph:
            with _lib.on_device(device):
                n = int(_lib.load().nsa_kv8_ticket_count())
            _graph[device.index] = [torch.zeros((_GRAPH_ROWS, n), dtype=torch.int32, device=device), 0]


def _capturing(index):
    """Whether the device's current stream is being captured."""
    if torch._C._cuda_getDevice() == index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _scratch(device, nbytes, stream):
    if _capturing(device.index):
        with _scratch_lock:
            rows, row = _graph[device.index]
            if row < rows.shape[0]:
                _graph[device.index][1] = row + 1
        tickets = rows[row] if row < rows.shape[0] else torch.zeros(rows.shape[1], dtype=torch.int32, device=device)
        return torch.empty(nbytes, dtype=torch.uint8, device=device), tickets
    pair = _eager.get((device.index, stream))
    if pair is None or pair[0].numel() < nbytes:
        with _scratch_lock:
            tickets = pair[1] if pair else torch.zeros_like(_graph[device.index][0][0])
            pair = _eager[(device.index, stream)] = (torch.empty(nbytes, dtype=torch.uint8, device=device), tickets)
    return pair


def _req(cond, msg, exc=ValueError):
    if not cond:
        raise exc(msg)


# Tensors that the kernels find by the address that the descriptor holds.
_STORAGE = frozenset(("k_codes", "v_codes", "scales", "page_table", "k_ring", "v_ring", "lens", "_ring_floor", "_unclean",
                      "_append_tickets"))


class Kv8CacheDesc(ctypes.Structure):
    """ctypes mirror of nsa_kv8_cache (include/nsa_b200.h)."""
    _fields_ = [(n, ctypes.c_int64) for n in ("batch", "n_kv_heads", "head_dim", "n_pages", "max_blocks")] + \
               [(n, ctypes.c_int32) for n in ("dtype", "codes")] + \
               [(n, ctypes.c_void_p) for n in ("k_codes", "v_codes", "scales", "page_table", "k_ring", "v_ring", "lens",
                                               "ring_floor", "unclean", "tickets")]


class Kv8Rows(ctypes.Structure):
    """ctypes mirror of nsa_kv8_rows."""
    _fields_ = [("data", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("batch_stride", "head_stride",
                                                                           "token_stride")]


class _RowArgs(threading.local):
    """nsa_kv8_rows of a call's tensors, one set a thread (making them anew costs 2 us each)."""

    def __init__(self):
        self.rows = [Kv8Rows() for _ in range(4)]
        self.refs = [ctypes.byref(r) for r in self.rows]


_row_args = _RowArgs()


def _rows(i, t, args=_row_args):
    """[B, H, D] or [B, H, T, D] as the call's i-th nsa_kv8_rows; dimensions of one element have no stride."""
    row, shape, st = args.rows[i], t.shape, t.stride()
    row.data = t.data_ptr()
    row.batch_stride = st[0] if shape[0] > 1 else 0
    row.head_stride = st[1] if shape[1] > 1 else 0
    row.token_stride = st[2] if len(shape) == 4 and shape[2] > 1 else 0
    return args.refs[i]


def _stream(index):
    """Raw handle of the device's current stream (a Stream object costs 2 us)."""
    return torch._C._cuda_getCurrentRawStream(index)


class Kv8Cache:
    """8-bit paged KV cache of one attention layer.

    ``batch`` sequences of up to ``max_len`` tokens.  ``n_pages`` None: every
    sequence has pages of its own; else a pool of that many pages, which the
    caller hands out by writing page numbers into ``page_table`` (int32
    [batch, blocks], initially 0) before a block is completed.  Sequences may
    share pages of complete blocks (``adopt``).  ``lens`` (int64 [batch]) holds
    the lengths, which the calls set; who writes one has to see to the ring's
    tokens of an incomplete block as well.

    Storage, readable at any time: ``k_codes`` / ``v_codes`` [n_pages, Hkv, 64,
    D] (float8_e4m3fn or int8), ``scales`` [n_pages, Hkv, 2] float32 (K, V),
    ``k_ring`` / ``v_ring`` [batch, Hkv, 128, D] (position p at slot p % 128).

    The table and the storage are written in place (``cache.page_table[b] =
    pages``); putting another tensor in the place of one is refused.

    Calls on one cache are ordered by their stream; calls that write (append,
    decode_step, truncate, adopt) must not overlap other calls on the cache.  A page
    number outside the pool, a length or start outside the table's room and a
    start that the ring no longer reaches are reported by ``device_error()``.
    """

    def __init__(self, batch, n_kv_heads, max_len, head_dim=D_HEAD, dtype=torch.float16, codes="e4m3", n_pages=None,
                 device=None):
        _req(head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}")
        _req(dtype in (torch.float16, torch.bfloat16), f"dtype must be float16 or bfloat16, got {dtype}", TypeError)
        _req(codes in _CODES, f"codes must be 'e4m3' or 'int8', got {codes!r}")
        batch, n_kv_heads, max_len = int(batch), int(n_kv_heads), int(max_len)
        _req(batch >= 0 and n_kv_heads > 0 and max_len > 0, "need batch >= 0, n_kv_heads > 0 and max_len > 0")
        _req(n_pages is None or n_pages >= 1, "n_pages must be positive")
        device = torch.device(device if device is not None else "cuda")
        _req(device.type == "cuda", "Kv8Cache lives on a CUDA device (no CPU fallback)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        _req(not _capturing(device.index), "a Kv8Cache cannot be made while a graph is captured", RuntimeError)
        self.batch, self.n_kv_heads, self.head_dim, self.dtype, self.codes = batch, n_kv_heads, head_dim, dtype, codes
        self.max_blocks = (max_len + BLOCK - 1) // BLOCK
        self.n_pages = max(1, batch * self.max_blocks) if n_pages is None else int(n_pages)
        self.device = device
        code, form = _CODES[codes]

        def z(shape, dt):
            return torch.zeros(shape, dtype=dt, device=device)

        page = (self.n_pages, n_kv_heads, BLOCK, head_dim)
        ring = (batch, n_kv_heads, RING, head_dim)
        self.k_codes, self.v_codes, self.scales = z(page, form), z(page, form), z(page[:2] + (2,), torch.float32)
        self.k_ring, self.v_ring = z(ring, dtype), z(ring, dtype)
        self.page_table = z((batch, self.max_blocks), torch.int32)
        if n_pages is None:
            self.page_table.copy_(torch.arange(batch * self.max_blocks, dtype=torch.int32).view(batch, self.max_blocks))
        self.lens, self._ring_floor = z((batch,), torch.int64), z((batch,), torch.int64)
        self._unclean, self._append_tickets = z((batch,), torch.int32), z((batch,), torch.int32)
        d = self._desc = Kv8CacheDesc(batch, n_kv_heads, head_dim, self.n_pages, self.max_blocks, _DTYPES[dtype], code)
        for n, t in (("k_codes", self.k_codes), ("v_codes", self.v_codes), ("scales", self.scales),
                     ("page_table", self.page_table), ("k_ring", self.k_ring), ("v_ring", self.v_ring),
                     ("lens", self.lens), ("ring_floor", self._ring_floor), ("unclean", self._unclean), ("tickets", self._append_tickets)):
            setattr(d, n, t.data_ptr())
        self._desc_ref = ctypes.byref(d)
        self._lib, self._index, self._ws_bytes = _lib.load(), device.index, {}
        _graph_rows(device)

    def __setattr__(self, name, value):
        if name in _STORAGE and self.__dict__.get(name, value) is not value:
            raise AttributeError(f"{name} is the cache's storage: write into it (indexing, copy_), it cannot be replaced")
        super().__setattr__(name, value)

    # ---------------------------------------------------------------- plumbing
    # (messages are built where they are raised: these checks run on every call)
    def _check(self, name, t, heads):
        """Checks [B, heads, D] or [B, heads, T, D] (heads 0: any multiple of the KV heads); returns T."""
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be a CUDA tensor on the cache's device {self.device} (no CPU fallback)")
        if t.dtype != self.dtype:
            raise TypeError(f"{name} must be {self.dtype}, got {t.dtype}")
        shape = t.shape
        n = len(shape)
        if not ((n == 3 or n == 4) and shape[0] == self.batch and shape[-1] == self.head_dim
                and (shape[1] == heads if heads else shape[1] > 0 and shape[1] % self.n_kv_heads == 0)):
            raise ValueError(f"{name} must be [{self.batch}, {heads or f'multiple of {self.n_kv_heads}'}, (T,) "
                             f"{self.head_dim}], got {tuple(shape)}")
        if t.stride(-1) != 1:
            raise ValueError(f"the last dimension of {name} must be contiguous")
        return shape[2] if n == 4 else 1

    def _words(self, name, t):
        """Device pointer of an optional int64 [B] tensor."""
        if t is None:
            return None
        if not (isinstance(t, torch.Tensor) and t.dtype == torch.int64 and t.get_device() == self._index
                and t.shape == (self.batch,) and t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int64 CUDA tensor of length B on the cache's device")
        return t.data_ptr()

    def _call(self, fn, *args):
        """fn(descriptor, *args, current stream of the cache's device), its status checked."""
        if torch._C._cuda_getDevice() == self._index:
            status = fn(self._desc_ref, *args, _stream(self._index))
        else:
            with torch.cuda.device(self._index):
                status = fn(self._desc_ref, *args, _stream(self._index))
        if status:
            _lib.check(status)

    def _scratch(self, heads, n_tokens):
        """Workspace and tickets of one attend."""
        nbytes = self._ws_bytes.get((heads, n_tokens))
        if nbytes is None:
            with _lib.on_device(self.device):  # (it depends on the device's number of SMs)
                nbytes = self._lib.nsa_kv8_workspace_bytes(self._desc_ref, heads, n_tokens)
            if self.batch and not nbytes:
                _lib.check(_lib.NSA_ERR_INVALID)  # raises with the library's message
            self._ws_bytes[heads, n_tokens] = nbytes
        return _scratch(self.device, nbytes, _stream(self._index))

    def _attend_args(self, sm_scale, window, sink):
        if window is not None and window < 0:
            raise ValueError("window must not be negative")
        window, sink = -1 if window is None else int(window), int(sink)
        if sink < 0:
            raise ValueError("sink must not be negative")
        return window, sink, self.head_dim ** -0.5 if sm_scale is None else float(sm_scale)

    # ---------------------------------------------------------------- writing
    def append(self, new_k, new_v, counts=None, starts=None):
        """Write new tokens behind each sequence's, quantizing every block that
        they complete.  new_k / new_v: [B, Hkv, D] or [B, Hkv, T, D] (any strides
        with the last dimension contiguous).  ``counts`` (int64 [B]): of the T
        tokens, how many each sequence takes; ``starts`` (int64 [B]): positions
        to write at instead of ``lens``, so that a start below it takes tokens
        back: to any multiple of 64, or as far as the block before the one in
        which the last append ended, but not into tokens that were adopted or
        lie below a multiple of 64 that was gone back to further than that."""
        t = self._check("new_k", new_k, self.n_kv_heads)
        if self._check("new_v", new_v, self.n_kv_heads) != t or new_v.dim() != new_k.dim():
            raise ValueError("new_k and new_v must have the same shape")
        self._call(self._lib.nsa_kv8_append, _rows(0, new_k), _rows(1, new_v), t, self._words("starts", starts),
                   self._words("counts", counts))

    def truncate(self, lens):
        """Set the lengths to ``lens`` (int64 [B]), taking tokens back as
        ``append``'s ``starts`` does (0 empties a sequence)."""
        _req(lens is not None, "lens must be a tensor")
        self._call(self._lib.nsa_kv8_append, None, None, 0, self._words("lens", lens), None)

    def adopt(self, lens):
        """Let sequence b begin with the ``lens[b]`` tokens (int64 [B], multiples
        of 64; -1 leaves it as it is) that the pages of its first blocks in
        ``page_table`` hold, written by another sequence.  Of these, only whole
        blocks can be taken back (give such a block a page of its own before it
        is written again)."""
        _req(lens is not None, "lens must be a tensor")
        self._call(self._lib.nsa_kv8_adopt, self._words("lens", lens))

    # ---------------------------------------------------------------- reading
    def read(self, n_tokens, starts=None, dtype=None):
        """The tokens at positions starts[b] (default 0) .. + n_tokens as attention
        sees them: (k, v) [B, Hkv, n_tokens, D] of ``dtype`` (float32, float16
        or bfloat16; default the cache's).  Positions outside a sequence are 0."""
        dtype = self.dtype if dtype is None else dtype
        _req(dtype in _DTYPES, f"dtype must be float32, float16 or bfloat16, got {dtype}", TypeError)
        n_tokens = int(n_tokens)
        _req(n_tokens >= 0, "n_tokens must not be negative")
        k, v = (torch.empty((self.batch, self.n_kv_heads, n_tokens, self.head_dim), dtype=dtype, device=self.device)
                for _ in range(2))
        self._call(self._lib.nsa_kv8_read, n_tokens, self._words("starts", starts), k.data_ptr(), v.data_ptr(),
                   _DTYPES[dtype])
        return k, v

    # ---------------------------------------------------------------- attention
    def attend(self, q, sm_scale=None, window=None, sink=SINK_SIZE, counts=None):
        """Attention of the sequences' last tokens -> o like q.

        q: [B, H, D], each sequence's last token, or [B, H, T, D] (T <= 64), its
        last T: row i stands at position lens - T + i and sees the tokens up to
        its own; with ``window`` only the newest ``window`` of them and the
        first ``sink``.  ``counts`` (int64 [B]): how many of the T query tokens
        each sequence has (row i then at lens - counts + i).  Rows that see
        nothing and rows behind counts are 0."""
        t, heads = self._check("q", q, 0), q.shape[1]
        window, sink, scale = self._attend_args(sm_scale, window, sink)
        o = torch.empty_like(q)
        ws, tickets = self._scratch(heads, t)
        self._call(self._lib.nsa_kv8_attend, _rows(0, q), _rows(1, o), heads, t, self._words("counts", counts), window,
                   sink, scale, ws.data_ptr(), ws.numel(), tickets.data_ptr())
        return o

    def decode_step(self, q, new_k, new_v, sm_scale=None, window=None, sink=SINK_SIZE, counts=None, starts=None):
        """append(new_k, new_v, counts, starts), then attend(q, ...) with the
        new tokens as queries: q [B, H, D] with new_k / new_v [B, Hkv, D], or
        all three with T tokens."""
        t, heads = self._check("q", q, 0), q.shape[1]
        if self._check("new_k", new_k, self.n_kv_heads) != t or self._check("new_v", new_v, self.n_kv_heads) != t:
            raise ValueError("q, new_k and new_v must hold the same number of tokens")
        window, sink, scale = self._attend_args(sm_scale, window, sink)
        o = torch.empty_like(q)
        ws, tickets = self._scratch(heads, t)
        self._call(self._lib.nsa_kv8_decode_step, _rows(0, new_k), _rows(1, new_v), _rows(2, q), _rows(3, o), heads, t,
                   self._words("starts", starts), self._words("counts", counts), window, sink, scale, ws.data_ptr(),
                   ws.numel(), tickets.data_ptr())
        return o
