"""A paged KV cache held in 8 bits, with the attention that reads it and
eviction by accumulated attention weight.

Beside PagedKVCache (bf16 / fp32, draftkv/paged.py:76-177 of the reference)
and CompressedKVCache (the drafter's slot arrays): half the bytes of the bf16
cache, the same block allocator and rollback, decode / verify / prompt
attention, and a bound on its length by eviction per KV head.  The reference
has no counterpart.

K and V are e4m3 codes under one power-of-two scale per block of tokens, KV
head and side (byte order: include/draftkv_b200.h, dkv_q8_cache).  Entries are
counted per layer from 0; until the first eviction entry i is position i.
"""

from __future__ import annotations

import numpy as np

from . import _lib
from .paged import BlockPoolExhausted, PagedKVCache

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

BLOCK_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_CODES = {} if torch is None else {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
MASS_ROWS = 64          # query rows a KV head up to which attention can add up the mass
WORK_ZERO_BYTES = 65536  # bytes at the start of an attention's scratch that are zero between calls


def tile_bytes(d_head: int):
    """(K, V) int64 tables [16, d]: the byte of element (token, dim) inside a
    16-token tile of the pool (the tensor core's operand order)."""
    tok, dim = np.arange(16)[:, None], np.arange(d_head)[None, :]
    blk, r, c = dim // 32, dim % 32, dim % 16
    k = blk * 512 + ((tok % 8) * 4 + (c % 8) // 2) * 16 + ((r // 16) * 2 + tok // 8) * 4 + (c // 8) * 2 + c % 2
    v = blk * 512 + ((c % 8) * 4 + (tok % 8) // 2) * 16 + ((r // 16) * 2 + c // 8) * 4 + (tok // 8) * 2 + tok % 2
    return k, v


def _check_i32(name: str, t, shape, device) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}")


class Q8KVCache(PagedKVCache):
    """The 8-bit paged cache: block tables and rollback of PagedKVCache, the
    pool in e4m3.  `track_mass` keeps per entry the softmax weight it has
    received (per layer [batch][n_kv][capacity], added to by attention calls
    and model forwards) and its position, which `evict` goes by."""

    def __init__(self, n_layers: int, n_heads: int, d_head: int, block_size: int = 16, n_blocks: int = 512,
                 batch: int = 1, max_blocks_per_seq: int | None = None, device: str = "cuda",
                 track_mass: bool = False) -> None:
        self._check_shape(d_head, block_size)
        self.track_mass = track_mass
        super().__init__(n_layers, n_heads, d_head, block_size=block_size, n_blocks=n_blocks, dtype=np.float32,
                         batch=batch, max_blocks_per_seq=max_blocks_per_seq, device=device)
        self.next_pos = [0] * batch          # position of the next token (entries + evicted)
        # per sequence and layer: entries from here on are the last positions of every head
        self._floor = [[0] * n_layers for _ in range(batch)]
        self._gone = [[0] * n_layers for _ in range(batch)]     # entries evicted since the sequence was empty

    @staticmethod
    def _check_shape(d_head: int, block_size: int) -> None:
        if d_head not in HEAD_DIMS:
            raise ValueError(f"the 8-bit cache holds heads of {HEAD_DIMS} (got {d_head})")
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"the 8-bit cache has blocks of {BLOCK_SIZES} tokens (got {block_size})")

    @classmethod
    def from_storage(cls, codes, scale, page_table, block_size: int = 16) -> "Q8KVCache":
        """A cache over storage the caller owns and allocates: codes uint8
        [n_pages, n_kv, 2, block_size * d], scale f32 [n_pages, n_kv, 2] and
        page_table int32 [batch, n_layers, max_pages], all contiguous on one
        CUDA device.  The device calls (write, attention, evict_rows, read_rows)
        work; the block allocator's methods do not."""
        if codes.dtype != torch.uint8 or codes.dim() != 4 or codes.shape[2] != 2 or not codes.is_contiguous():
            raise ValueError("codes must be a contiguous uint8 tensor [n_pages, n_kv, 2, block_size * d]")
        if codes.shape[3] % block_size:
            raise ValueError(f"codes rows of {codes.shape[3]} bytes are no whole block of {block_size} tokens")
        self = cls.__new__(cls)
        self.n_heads, self.d_head = codes.shape[1], codes.shape[3] // block_size
        cls._check_shape(self.d_head, block_size)
        if scale.dtype != torch.float32 or tuple(scale.shape) != tuple(codes.shape[:3]) or not scale.is_contiguous():
            raise ValueError("scale must be a contiguous float32 tensor [n_pages, n_kv, 2]")
        if page_table.dtype != torch.int32 or page_table.dim() != 3 or not page_table.is_contiguous():
            raise ValueError("page_table must be a contiguous int32 tensor [batch, n_layers, max_pages]")
        if not (codes.is_cuda and scale.device == codes.device and page_table.device == codes.device):
            raise ValueError("codes, scale and page_table must be on one CUDA device")
        self.batch, self.n_layers, self.max_pages = page_table.shape
        self.block_size, self.device, self.track_mass = block_size, codes.device, False
        self.pool, self.mass, self.pos_t = None, None, None
        self.codes, self.scale, self.table_dev = codes, scale, page_table
        self._dirty = False
        self._finish_struct()
        return self

    # ------------------------------------------------------------ device
    def _alloc_device(self, n_blocks: int) -> None:
        _lib.load()
        dev = self.device
        self.codes = torch.zeros((n_blocks, self.n_heads, 2, self.block_size * self.d_head), dtype=torch.uint8, device=dev)
        self.scale = torch.ones((n_blocks, self.n_heads, 2), dtype=torch.float32, device=dev)
        self.table_host = torch.zeros((self.batch, self.n_layers, self.max_pages), dtype=torch.int32, pin_memory=True)
        self.table_dev = torch.zeros((self.batch, self.n_layers, self.max_pages), dtype=torch.int32, device=dev)
        self.device = self.codes.device
        self._dirty = False
        shape = (self.batch, self.n_heads, self.max_pages * self.block_size)
        self.mass = self.pos_t = None
        if self.track_mass:
            # one more than the layers: eviction writes out of place and swaps
            self.mass = [torch.zeros(shape, dtype=torch.float32, device=dev) for _ in range(self.n_layers + 1)]
            self.pos_t = [torch.full(shape, -1, dtype=torch.int32, device=dev) for _ in range(self.n_layers + 1)]
        self._finish_struct()

    def _finish_struct(self) -> None:
        self._struct = _lib.Q8CacheS(self.codes.data_ptr(), self.scale.data_ptr(), self.table_dev.data_ptr(),
                                     self.codes.shape[0], self.block_size, self.max_pages)
        self._dims = _lib.DimsS(self.n_layers, self.n_heads, self.d_head, self.batch)
        self._work: dict = {}            # scratch by stream (threads with streams of their own do not meet)
        self._work_bytes: dict = {}      # its size by call

    def struct(self) -> "_lib.Q8CacheS":
        self.sync_table()
        return self._struct

    def layer_arrays(self):
        """Device addresses of the layers' mass and positions (empty: not kept)."""
        if not self.track_mass or self.mass is None:
            return (), ()
        return tuple(t.data_ptr() for t in self.mass[:-1]), tuple(t.data_ptr() for t in self.pos_t[:-1])

    @property
    def host_resident(self) -> bool:
        return False

    def offload_to_host(self) -> None:
        raise NotImplementedError("the 8-bit cache stays in device memory")

    @property
    def nbytes(self) -> int:
        """Bytes of the pool (codes and scales)."""
        return self.codes.numel() + self.scale.numel() * 4

    def _workspace(self, T: int, group: int, split_keys: int, note_mass: bool, stream: int):
        """The attention scratch of a call: one buffer per stream (calls on one
        stream run in order), grown to the largest call; its tickets are zero
        when made and left so by each call.  A call that is being captured gets
        one of its own, cleared by the graph itself: graphs may be replayed side
        by side."""
        key = (T, group, split_keys, note_mass)
        n = self._work_bytes.get(key)
        if n is None:
            n = max(int(_lib.load().dkv_q8_attn_work_bytes(self._dims, group, T, self.capacity_tokens, split_keys,
                                                           1 if note_mass else 0)), WORK_ZERO_BYTES)
            self._work_bytes[key] = n
        capturing = torch.cuda.is_current_stream_capturing()
        w = None if capturing else self._work.get(stream)
        if w is None or w.numel() < n:
            w = torch.empty(n, dtype=torch.uint8, device=self.device)
            w[:WORK_ZERO_BYTES].zero_()
            if not capturing:            # (the smaller one goes)
                self._work[stream] = w
        return w

    def _stream(self) -> int:
        """The current stream, of the cache's device (which has to be the current
        one: launches go there)."""
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the cache is on {self.device}, the current device is cuda:{torch.cuda.current_device()}")
        return _lib.stream_ptr()

    # ------------------------------------------------------ device calls
    def write(self, layer: int, k, v, entry0, n_rows=None, pos0=None, mass=None, pos=None) -> None:
        """Quantizes rows into entries entry0[b] .. of `layer` on the device.
        k, v: [batch, rows, n_kv, d] bf16 or fp32, any strides with the last
        dimension contiguous (the same for both); entry0, n_rows, pos0: int32
        [batch].  mass / pos ([batch, n_kv, capacity]): reset for the new
        entries.  The pages must be in the table (`ensure`)."""
        stream, shape, strides, code = self._stream(), k.shape, k.stride(), _CODES.get(k.dtype)
        if len(shape) != 4 or shape[0] != self.batch or shape[2] != self.n_heads or shape[3] != self.d_head:
            raise ValueError(f"k must be [{self.batch}, rows, {self.n_heads}, {self.d_head}], got {tuple(shape)}")
        if v.shape != shape or v.dtype is not k.dtype or v.stride() != strides:
            raise ValueError("k and v must have one shape, dtype and strides")
        if k.device != self.device or v.device != self.device:
            raise ValueError(f"k and v must be on {self.device}")
        if code is None or strides[3] != 1:
            raise ValueError("k and v must be bf16 or fp32 with a contiguous last dimension")
        _check_i32("entry0", entry0, (self.batch,), self.device)
        for name, t in (("n_rows", n_rows), ("pos0", pos0)):
            if t is not None:
                _check_i32(name, t, (self.batch,), self.device)
        self._check_mass(mass)
        if pos is not None:
            _check_i32("pos", pos, self._mass_shape(), self.device)
        rows = shape[1]
        if rows == 0:
            return
        _lib.call("dkv_q8_append", self.struct(), self._dims, layer, k.data_ptr(), v.data_ptr(), code, rows, strides[0],
                  strides[1], strides[2], entry0.data_ptr(), _lib.ptr(n_rows), _lib.ptr(pos0), _lib.ptr(mass),
                  _lib.ptr(pos), stream)

    def _mass_shape(self):
        return (self.batch, self.n_heads, self.capacity_tokens)

    def _check_mass(self, mass) -> None:
        if mass is not None and (mass.dtype is not torch.float32 or mass.shape != self._mass_shape()
                                 or not mass.is_contiguous() or mass.device != self.device):
            raise ValueError(f"mass must be a contiguous float32 tensor of shape {self._mass_shape()} on {self.device}")

    def attention(self, layer: int, q, entry0, n_rows=None, mass=None, out=None, out_dtype=None, split_keys: int = 0,
                  work=None):
        """Causal attention of q [batch, T, n_heads, d] fp32 over `layer`: token
        t of sequence b sees entries 0 .. entry0[b] + t (those of the call must
        have been written).  Returns [batch, T, n_heads, d] in out_dtype (bf16
        by default); tokens t >= n_rows[b] are skipped and their rows of `out`
        left as they were (zeros when `out` is made here).  mass (T * n_heads /
        n_kv <= 64): every seen entry's softmax weights are added to it.  A row
        of up to 64 equals the one-token call at that entry bit for bit.  With
        fp32 outputs queries and weights keep 22 bits; with bf16 outputs weights
        keep 11, and queries too where T * n_heads / n_kv > 64.  `work`:
        uint8 scratch of `dkv_q8_attn_work_bytes`, the first 64 KB zero when
        first used, for a caller that keeps its own; by default the cache has one
        per stream, and a captured call one of its own."""
        stream, shape, kv = self._stream(), q.shape, self.n_heads
        if len(shape) != 4 or shape[0] != self.batch or shape[3] != self.d_head or shape[2] % kv or not shape[2]:
            raise ValueError(f"q must be [{self.batch}, T, a multiple of {kv} heads, {self.d_head}], got {tuple(shape)}")
        if q.dtype is not torch.float32 or q.device != self.device or not q.is_contiguous():
            raise ValueError(f"q must be a contiguous float32 tensor on {self.device}")
        _check_i32("entry0", entry0, (self.batch,), self.device)
        if n_rows is not None:
            _check_i32("n_rows", n_rows, (self.batch,), self.device)
        self._check_mass(mass)
        T, group = shape[1], shape[2] // kv
        if out is None:
            make = torch.empty_like if n_rows is None else torch.zeros_like
            out = make(q, dtype=out_dtype or torch.bfloat16)
        elif out.shape != shape or not out.is_contiguous() or out.device != self.device \
                or (out_dtype is not None and out.dtype is not out_dtype):
            raise ValueError("out must be contiguous and shaped like q")
        code = _CODES.get(out.dtype)
        if code is None:
            raise ValueError("attention writes bf16 or fp32")
        if T == 0:
            return out
        if work is None:
            work = self._workspace(T, group, split_keys, mass is not None, stream)
        elif work.dtype is not torch.uint8 or work.device != self.device or not work.is_contiguous():
            raise ValueError(f"work must be a contiguous uint8 tensor on {self.device}")
        _lib.call("dkv_q8_attn", self.struct(), self._dims, layer, group, T, q.data_ptr(), entry0.data_ptr(),
                  _lib.ptr(n_rows), out.data_ptr(), code, split_keys, _lib.ptr(mass), work.data_ptr(), work.numel(), stream)
        return out

    def evict_rows(self, layer: int, n, budget, out_table, mass, pos=None, sink: int = 0, recent: int = 0,
                   mass_out=None, pos_out=None):
        """Per (sequence, KV head), of the first n[b] entries of `layer` keeps
        min(n, max(budget[b], sink + recent)): the first `sink`, the last
        `recent` and those of the most mass (the lowest (mass, index) are
        dropped).  They are written to the pages out_table [batch, out_pages],
        which must be in no row of the page table.  Returns (kept [batch, n_kv,
        out_pages * block_size] int32 entry indices, -1 behind; mass_out;
        pos_out or None)."""
        stream = self._stream()
        _check_i32("n", n, (self.batch,), self.device)
        _check_i32("budget", budget, (self.batch,), self.device)
        if out_table.dim() != 2:
            raise ValueError("out_table must be [batch, out_pages]")
        _check_i32("out_table", out_table, (self.batch, out_table.shape[1]), self.device)
        if mass is None:
            raise ValueError("eviction goes by the attention mass")
        self._check_mass(mass)
        self._check_mass(mass_out)
        for name, t in (("pos", pos), ("pos_out", pos_out)):
            if t is not None:
                _check_i32(name, t, self._mass_shape(), self.device)
        if mass_out is None:
            mass_out = torch.empty_like(mass)
        if pos is None:
            pos_out = None
        elif pos_out is None:
            pos_out = torch.empty_like(pos)
        out_pages = out_table.shape[1]
        kept = out_table.new_empty((self.batch, self.n_heads, out_pages * self.block_size))
        _lib.call("dkv_q8_evict", self.struct(), self._dims, layer, n.data_ptr(), budget.data_ptr(), sink, recent,
                  mass.data_ptr(), _lib.ptr(pos), out_table.data_ptr(), out_pages, mass_out.data_ptr(), _lib.ptr(pos_out),
                  kept.data_ptr(), stream)
        return kept, mass_out, pos_out

    def read_rows(self, layer: int, n: int, b: int = 0):
        """Entries [0, n) of one sequence, dequantized: fp32 [n, n_kv, 2, d] on
        the device."""
        stream = self._stream()
        out = torch.empty((n, self.n_heads, 2, self.d_head), dtype=torch.float32, device=self.device)
        _lib.call("dkv_q8_read", self.struct(), self._dims, b, layer, n, out.data_ptr(), stream)
        return out

    # ---------------------------------------------------- cache protocol
    def append(self, layer: int, k, v, pos) -> None:
        """Rows (numpy [rows, n_kv, d]) of sequence 0 at its end; positions must
        go on where the layer's end (after an eviction ahead of the entries)."""
        k, v = np.asarray(k, np.float32), np.asarray(v, np.float32)
        pos = np.asarray(pos).reshape(-1)
        n, start = k.shape[0], self.counts[0][layer]
        if n == 0:
            return
        if not np.array_equal(pos, start + self._gone[0][layer] + np.arange(n)):
            raise ValueError("appended positions must be consecutive and continue the cache's")
        self._ensure_layer(0, layer, start + n)
        kv = torch.from_numpy(np.ascontiguousarray(np.stack([k, v])[:, None])).to(self.device)
        rows = torch.zeros((self.batch,), dtype=torch.int32)
        rows[0] = n
        e0 = torch.zeros((self.batch,), dtype=torch.int32)
        e0[0] = start
        p0 = torch.full((self.batch,), int(pos[0]), dtype=torch.int32, device=self.device)
        kv = kv.expand(2, self.batch, -1, -1, -1)
        self.write(layer, kv[0], kv[1], e0.to(self.device), n_rows=rows.to(self.device), pos0=p0,
                   mass=self.mass[layer] if self.mass else None, pos=self.pos_t[layer] if self.pos_t else None)
        self.counts[0][layer] = start + n
        if layer == 0:
            self.next_pos[0] = int(pos[0]) + n

    def _ensure_layer(self, b: int, layer: int, n_tokens: int) -> None:
        need = -(-n_tokens // self.block_size)
        if need > self.max_pages:
            raise BlockPoolExhausted(f"sequence needs {need} blocks > max_blocks_per_seq {self.max_pages}")
        tbl = self.block_tables[b][layer]
        if len(tbl) < need:
            new = self.pool.allocate_many(need - len(tbl))
            self.table_host[b, layer, len(tbl):need] = torch.tensor(new, dtype=torch.int32)
            tbl.extend(new)
            self._dirty = True

    def positions(self, layer: int, b: int = 0):
        """Positions [n_kv, entries] of a sequence's entries (numpy int64)."""
        n = self.counts[b][layer]
        if self.pos_t is None:
            return np.broadcast_to(np.arange(n, dtype=np.int64), (self.n_heads, n))
        return self.pos_t[layer][b, :, :n].cpu().numpy().astype(np.int64)

    def read(self, layer: int, b: int = 0):
        """Dequantized (k, v, positions) of a sequence's entries.  Positions are
        [entries] while every head holds the same ones, [n_kv, entries] after an
        eviction that parted them."""
        n = self.counts[b][layer]
        if n == 0:
            z = np.zeros((0, self.n_heads, self.d_head), np.float32)
            return z, z.copy(), np.zeros((0,), np.int64)
        o = self.read_rows(layer, n, b).cpu().numpy()
        pos = self.positions(layer, b)
        return o[:, :, 0], o[:, :, 1], pos[0] if (pos == pos[:1]).all() else pos

    @property
    def pos(self):
        """Positions of sequence 0's entries per layer, as `read` gives them."""
        each = (self.positions(L) for L in range(self.n_layers))
        return [(p[0] if (p == p[:1]).all() else p).tolist() for p in each]

    def truncate_seq(self, b: int, n_pos: int) -> None:
        """Rollback to n_pos entries (paged.py:144-162); the scale of a partly
        emptied block stays until the block is written from its start again.
        After an eviction a sequence can go back through its recent entries (or
        to none): before them the heads hold different positions.  Layers of
        which different numbers were evicted can only go back together while
        they hold equally many entries: otherwise entry n_pos is another position
        in each."""
        n_pos, counts = max(n_pos, 0), self.counts[b]
        self._check_rollback(b, n_pos)
        if n_pos >= max(counts):
            return
        if n_pos == 0:
            self._floor[b], self._gone[b] = [0] * self.n_layers, [0] * self.n_layers
        before = counts[0]
        super().truncate_seq(b, n_pos)
        left = counts[0]
        self.next_pos[b] = self.next_pos[b] - (before - left) if left else 0

    def _check_rollback(self, b: int, n_pos: int) -> None:
        counts, floor = self.counts[b], max(self._floor[b])
        if not 0 < n_pos < max(counts):
            return
        if len(set(counts)) > 1 and len(set(self._gone[b])) > 1:
            raise ValueError(f"the layers of sequence {b} hold different positions (evict all of them alike)")
        if n_pos < floor:
            raise ValueError(f"entries before {floor} of sequence {b} hold other positions in each head")

    def truncate(self, n_pos: int) -> None:
        """Every sequence, or where one cannot go back to n_pos none."""
        for b in range(self.batch):
            self._check_rollback(b, n_pos)
        super().truncate(n_pos)

    def set_length(self, b: int, n: int) -> None:
        self.next_pos[b] += n - self.counts[b][0]
        super().set_length(b, n)

    def evict(self, budget: int, sink: int = 4, recent: int = 16, layers=None):
        """Prunes every sequence to at most max(budget, sink + recent) entries a
        layer by accumulated attention mass, per KV head.  New blocks are taken
        from the pool before the old ones return to it (BlockPoolExhausted leaves
        the cache as it was; where a call fails later, the layers before it are
        pruned, and it and those behind it are as they were).  Returns {layer: kept entry indices [batch, n_kv,
        .] on the device} of the layers that were pruned."""
        if not self.track_mass:
            raise ValueError("evict needs track_mass=True")
        if budget < 1 or sink < 0 or recent < 0:
            raise ValueError("evict: budget >= 1, sink >= 0, recent >= 0")
        keep_to = max(budget, sink + recent)
        self._stream()
        plan, free = [], self.pool.n_free
        for L in dict.fromkeys(range(self.n_layers) if layers is None else layers):
            if not 0 <= L < self.n_layers:
                raise ValueError(f"evict: layer {L} of {self.n_layers}")
            n = [self.counts[b][L] for b in range(self.batch)]
            if max(n) <= keep_to:
                continue
            m = [min(x, keep_to) for x in n]
            pages = [-(-x // self.block_size) for x in m]
            if sum(pages) > free:
                raise BlockPoolExhausted(f"eviction needs {sum(pages)} free blocks, {free} left")
            free += sum(len(self.block_tables[b][L]) for b in range(self.batch)) - sum(pages)
            plan.append((L, n, m, pages))
        out = {}
        for L, n, m, pages in plan:
            new = [self.pool.allocate_many(p) for p in pages]
            try:
                table = torch.full((self.batch, max(max(pages), 1)), -1, dtype=torch.int32)
                for b, ids in enumerate(new):
                    table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
                dev = self.device
                out[L], _, _ = self.evict_rows(
                    L, torch.tensor(n, dtype=torch.int32).to(dev), torch.tensor(m, dtype=torch.int32).to(dev), table.to(dev),
                    self.mass[L], self.pos_t[L], sink, recent, self.mass[-1], self.pos_t[-1])
            except BaseException:
                for blk in reversed([blk for ids in new for blk in ids]):
                    self.pool.free(blk)
                raise
            self.mass[L], self.mass[-1] = self.mass[-1], self.mass[L]
            self.pos_t[L], self.pos_t[-1] = self.pos_t[-1], self.pos_t[L]
            for b, ids in enumerate(new):
                for blk in reversed(self.block_tables[b][L]):
                    self.pool.free(blk)
                self.block_tables[b][L] = list(ids)
                self.table_host[b, L, :len(ids)] = table[b, :len(ids)]
                self.counts[b][L] = m[b]
                if n[b] > m[b]:
                    self._gone[b][L] += n[b] - m[b]
                    self._floor[b][L] = max(self._floor[b][L] - (n[b] - m[b]), m[b] - recent)
            self._dirty = True
        return out
