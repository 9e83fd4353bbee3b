"""The key/value store held in 4 bits, over the C ABI's b2_store_*: rows written into it, read back, and the arrival
(attention) over it.

    from streaming_machine_b200 import convert, store
    st = store.Store(convert.tables(), n_streams=64, max_ctx=1024, n_head=12)
    st.write(k, v, pos)              # one new position per stream: k, v [64, 12, 64] int64, pos [64] int32
    y = st.attend(q, pos)            # [64, 12, 64] int64: what each row takes from its stream's positions 0 .. pos
    y = st.step(q, k, v, pos)        # both in one launch
    k4, v4 = st.read(pos)            # the values that the store holds for those positions

Numbers are whole, at the stream's scale 2^-16; include/base2.h has the formulas. A prompt pass gives many rows per
stream: stream i's are rows cu[i] .. cu[i + 1] - 1, its first at position pos[i], none with more than max_rows.
Tensors are CUDA tensors of the store's device; calls queue their work on the current stream, allocate nothing but what
they return and copy nothing to the host, so that they may be captured into a graph.
"""
from __future__ import annotations

import ctypes

import numpy as np

from .engine import B2Error, StoreConfig, _torch, lib

HEAD = 64
INT32_MIN, INT32_MAX = -2 ** 31, 2 ** 31 - 1
_ended = []      # (handle, memory) of stores that ended while a graph was captured: freeing one waits for the device


def _free_ended(torch):
    """Free what has ended, unless a capture is under way on this thread's stream (the wait would break it)."""
    while _ended and not torch.cuda.is_current_stream_capturing():
        try:
            h, memory = _ended.pop()
        except IndexError:                               # another thread has taken the last
            return
        lib().b2_store_destroy(h)                        # (waits for the device: the memory may be used again)
        del memory


def _i32(x: int) -> int:
    """A number as the C ABI's int32 takes it: one outside stands for the nearest (ctypes would drop its upper bits). The
    calls come here where x >> 31 is not 0."""
    return x if INT32_MIN <= x <= INT32_MAX else (INT32_MIN if x < 0 else INT32_MAX)


class Store:
    """A 4-bit key/value store of `n_streams` streams of up to `max_ctx` positions, with `n_head` heads of 64 dims in each
    of `n_layer` layers; every position stands for zeros until it is written. M: the machine's tables ("arrival", "log2",
    "exp2", as convert.tables() or a converted model holds them). Making one waits for the device: not during a capture.

    What the streams hold is known on the device alone, so attend() and step() choose how a call is launched by max_ctx (or
    the window, where that is less): give a store about the context that its streams will reach. 512 streams of up to 192
    positions take 17 us in a store of 192 or 1,024, 62 in one of 2,048 and 487 in one of 32,768."""

    def __init__(self, M: dict, n_streams: int, max_ctx: int, n_head: int, n_layer: int = 1, device: int = 0):
        self.h = None
        self._host(_torch(), "cuda", device, n_streams, max_ctx, n_head, n_layer)
        _free_ended(self.torch)
        t = [np.ascontiguousarray(M[k], dtype=np.int64) for k in ("arrival", "log2", "exp2")]
        if t[1].size != 65536 or t[2].size != 65536:
            raise ValueError("the log2 and exp2 tables have 65,536 entries")
        h = ctypes.c_void_p()
        cfg = StoreConfig(*(_i32(x) for x in (n_streams, n_layer, n_head, max_ctx)))
        size = lib().b2_store_size(ctypes.byref(cfg), t[0].size)
        # torch's allocator gives the memory (and keeps it between stores)
        self._memory = self.torch.empty(max(size, 0), dtype=self.torch.uint8, device=self.device)
        rc = lib().b2_store_create(ctypes.byref(cfg), device, t[0].ctypes.data, t[0].size, t[1].ctypes.data, t[2].ctypes.data,
                                   self._memory.data_ptr(), ctypes.byref(h))
        self.h = h if h.value else None
        if rc:
            msg = lib().b2_store_last_error(self.h).decode() if self.h else f"b2_store_create failed ({n_streams} streams, " \
                f"{n_layer} layers, {n_head} heads, context {max_ctx}, device {device})"
            self.close()
            raise B2Error(rc, msg)

    def _host(self, torch, kind: str, device: int, n_streams: int, max_ctx: int, n_head: int, n_layer: int):
        """The host side's own state (no device work)."""
        cuda = kind == "cuda"
        self.torch, self.device = torch, torch.device(kind, device if cuda else None)
        self.n_streams, self.max_ctx, self.n_head, self.n_layer = n_streams, max_ctx, n_head, n_layer
        self._tensor, self._i64, self._i32 = torch.Tensor, torch.int64, torch.int32
        self._row, self._flat, self._unit = (n_head, HEAD), (n_head * HEAD,), (HEAD, 1)
        self._width = n_head * HEAD
        self._none = torch.empty(0, dtype=torch.int64, device=self.device)
        self._stream, self._index = (torch._C._cuda_getCurrentRawStream, device) if cuda else (lambda i: None, -1)
        L = lib()
        self._f_write, self._f_read, self._f_attend, self._f_step = L.b2_store_write, L.b2_store_read, L.b2_store_attend, L.b2_store_step

    # ---- plumbing ---------------------------------------------------------------------------------------------
    # (a decode step comes here for every layer: the usual case is settled by a few comparisons, what is wrong with an
    # argument is looked for only where they fail)
    def _rows(self, x, name: str):
        """(pointer, row stride) of int64 rows [rows, n_head, 64] or [rows, n_head * 64]; only the rows may be strided."""
        if isinstance(x, self._tensor) and x.dtype is self._i64 and x.get_device() == self._index:
            if x.ndim == 3 and x.is_contiguous():
                _, h, d = x.shape
                if h == self.n_head and d == HEAD:
                    return x.data_ptr(), self._width
            shape, st, d = x.shape, x.stride(), self._width
            if (shape[1:] == self._row and (st[1:] == self._unit or (self.n_head == 1 and st[2] == 1))) or \
                    (shape[1:] == self._flat and st[1] == 1):
                if st[0] >= d:
                    return x.data_ptr(), st[0]
                if shape[0] <= 1:                                # a single row's stride says nothing
                    return x.data_ptr(), d
            if shape[:1] == (0,) and shape[1:] in (self._row, self._flat):
                return x.data_ptr(), d                           # no rows: no stride says anything
            raise ValueError(f"{name}: rows of [{self.n_head}, {HEAD}] (or {d}) values, one behind the other and apart, got "
                             f"shape {tuple(shape)}, strides {st}")
        raise ValueError(f"{name}: a torch.int64 tensor on {self.device}, got {self._what(x)}")

    def _what(self, x) -> str:
        return f"{x.dtype} on {x.device}" if isinstance(x, self._tensor) else type(x).__name__

    def _ints(self, x, name: str, n: int):
        if isinstance(x, self._tensor) and x.dtype is self._i32 and x.get_device() == self._index and x.ndim == 1 and \
                x.numel() == n and x.is_contiguous():
            return x.data_ptr()
        what = f"shape {tuple(x.shape)}, strides {x.stride()}, " if isinstance(x, self._tensor) else ""
        raise ValueError(f"{name}: {n} torch.int32 values in a row on {self.device}, got {what}{self._what(x)}")

    def _table(self, pos, cu, rows: int, max_rows):
        """The row table's arguments: cu, pos, n_streams, rows, max_rows."""
        n = pos.numel() if isinstance(pos, self._tensor) else -1
        p = self._ints(pos, "pos", n)
        if cu is not None:
            if max_rows is None:
                raise ValueError("max_rows (the most rows a stream gives) goes with cu")
            c = self._ints(cu, "cu", n + 1)
            if (n | max_rows) >> 31:
                n, max_rows = _i32(n), _i32(max_rows)
            return c, p, n, rows, max_rows
        if rows != n or max_rows not in (None, 1):
            raise ValueError(f"without cu every stream gives one row: {rows} rows, {n} positions, max_rows {max_rows}")
        return None, p, n, rows, 1

    def _out(self, out, rows: int, name: str):
        shape = (rows, *self._row)
        if isinstance(out, self._tensor) and out.dtype is self._i64 and out.get_device() == self._index and \
                out.shape == shape and out.is_contiguous():
            return out
        what = f"shape {tuple(out.shape)}, strides {out.stride()}, " if isinstance(out, self._tensor) else ""
        raise ValueError(f"{name}: a contiguous {shape} of torch.int64 on {self.device}, got {what}{self._what(out)}")

    def _done(self, rc: int):
        if rc:
            raise B2Error(rc, lib().b2_store_last_error(self.h).decode())

    def _open(self):
        if not self.h:
            raise ValueError("the store is closed")
        return self.h

    # ---- the operators ----------------------------------------------------------------------------------------
    def write(self, k, v, pos, cu=None, max_rows: int | None = None, layer: int = 0):
        """Hold rows k, v (int64 [rows, n_head, 64], or rows of n_head * 64; rows may be strided, as slices of a qkv row
        are) at their streams' positions. A stream's rows that do not fit the call or the context are skipped (sync())."""
        h = self._open()
        if layer >> 31:
            layer = _i32(layer)
        (pk, ldk), (pv, ldv), rows = self._rows(k, "k"), self._rows(v, "v"), k.shape[0]
        if rows != v.shape[0]:
            raise ValueError(f"{rows} rows of keys, {v.shape[0]} of values")
        cu, pos, n, rows, most = self._table(pos, cu, rows, max_rows)
        rc = self._f_write(h, layer, pk, ldk, pv, ldv, cu, pos, n, rows, most, self._stream(self._index))
        if rc:
            self._done(rc)

    def read(self, pos, cu=None, max_rows: int | None = None, rows: int | None = None, layer: int = 0, out=None):
        """(k, v), int64 [rows, n_head, 64]: the values that the store holds at the rows' positions. rows: how many there
        are (with cu; its last entry). out: two tensors to fill instead of new ones. Rows that no stream has keep what
        `out` held (without it, uninitialised memory)."""
        h = self._open()
        if layer >> 31:
            layer = _i32(layer)
        if rows is None:
            if cu is not None:
                raise ValueError("rows (cu's last entry) goes with cu")
            rows = pos.numel() if isinstance(pos, self._tensor) else len(pos)
        if out is None:
            k = self._none.new_empty((rows, *self._row))     # (quicker than torch.empty, or one tensor taken apart)
            v = self.torch.empty_like(k)
        else:
            k, v = self._out(out[0], rows, "out k"), self._out(out[1], rows, "out v")
        cu, pos, n, rows, most = self._table(pos, cu, rows, max_rows)
        rc = self._f_read(h, layer, cu, pos, n, rows, most, k.data_ptr(), v.data_ptr(), self._stream(self._index))
        if rc:
            self._done(rc)
        return k, v

    def attend(self, q, pos, cu=None, max_rows: int | None = None, window: int = 0, first=None, layer: int = 0, out=None):
        """The arrival of rows q (int64 [rows, n_head, 64], or rows of n_head * 64, strided or not) over the held keys and
        values: int64 [rows, n_head, 64]. A row at position p sees the positions from the largest of 0, first[stream] (if
        given) and p - window + 1 (if window > 0) to p; one that sees none gets zeros. Rows that no stream has, and those of a
        stream that a device check skips (sync()), keep what `out` held: without `out` that is uninitialised memory."""
        h = self._open()
        if (layer | window) >> 31:
            layer, window = _i32(layer), _i32(window)
        pq, ldq = self._rows(q, "q")
        rows = q.shape[0]
        if out is not None:
            out = self._out(out, rows, "out")
        elif q.dim() == 3 and q.is_contiguous():
            out = self.torch.empty_like(q)               # (the quickest)
        else:
            out = q.new_empty((rows, *self._row))
        cu, pos, n, rows, most = self._table(pos, cu, rows, max_rows)
        f = None if first is None else self._ints(first, "first", n)
        rc = self._f_attend(h, layer, pq, ldq, cu, pos, f, n, rows, most, window, out.data_ptr(), self._stream(self._index))
        if rc:
            self._done(rc)
        return out

    def step(self, q, k, v, pos, window: int = 0, first=None, layer: int = 0, out=None):
        """A decode step, write() and attend() of one row a stream in one launch: row i is stream i's, at position pos[i].
        Where a stream between others has ended, write() and attend() with a cu that gives it no row do the same."""
        h = self._open()
        if (layer | window) >> 31:
            layer, window = _i32(layer), _i32(window)
        (pq, ldq), (pk, ldk), (pv, ldv), n = self._rows(q, "q"), self._rows(k, "k"), self._rows(v, "v"), q.shape[0]
        if k.shape[0] != n or v.shape[0] != n:
            raise ValueError(f"{n} rows of queries, {k.shape[0]} of keys, {v.shape[0]} of values")
        if out is not None:
            out = self._out(out, n, "out")
        elif q.dim() == 3 and q.is_contiguous():
            out = self.torch.empty_like(q)
        else:
            out = q.new_empty((n, *self._row))
        p = self._ints(pos, "pos", n)
        f = None if first is None else self._ints(first, "first", n)
        rc = self._f_step(h, layer, pq, ldq, pk, ldk, pv, ldv, p, f, n, window, out.data_ptr(), self._stream(self._index))
        if rc:
            self._done(rc)
        return out

    def sync(self):
        """Wait for the device and raise what its checks flagged (rows that do not fit the call, a position past the
        context): the streams concerned were skipped."""
        self._done(lib().b2_store_sync(self._open()))

    def close(self):
        """Free the store once the device is done with it. During a capture on this thread's stream that is put off until a
        store is made or closed outside of one (a capture in another thread is not seen: end no store meanwhile)."""
        if getattr(self, "h", None):
            _ended.append((self.h, self._memory))
            self.h = self._memory = None
            _free_ended(self.torch)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
