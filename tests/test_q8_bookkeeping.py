"""Which entries and positions an 8-bit cache holds, layer by layer: appends,
rollbacks, evictions and their failures, with the device calls replaced by host
ones (no GPU)."""
import copy

import numpy as np
import pytest

from tests import q8_reference as ref

torch = pytest.importorskip("torch")
from draftkv import BlockPoolExhausted, Q8KVCache  # noqa: E402


class HostCache(Q8KVCache):
    """Q8KVCache whose kernels run on the host: rows are not stored, positions and masses are."""
    fail = False

    def __init__(self, n_layers=2, batch=1, n_blocks=40, max_blocks=16):
        super().__init__(n_layers, 2, 64, block_size=16, n_blocks=n_blocks, batch=batch, max_blocks_per_seq=max_blocks,
                         device="cpu", track_mass=True)

    def _alloc_device(self, n_blocks):
        self.table_host = torch.zeros((self.batch, self.n_layers, self.max_pages), dtype=torch.int32)
        self._dirty = False
        shape = (self.batch, self.n_heads, self.max_pages * self.block_size)
        g = torch.Generator().manual_seed(0)
        self.mass = [torch.rand(shape, generator=g) for _ in range(self.n_layers + 1)]
        self.pos_t = [torch.full(shape, -1, dtype=torch.int32) for _ in range(self.n_layers + 1)]

    def _stream(self):
        return 0

    def write(self, layer, k, v, entry0, n_rows=None, pos0=None, mass=None, pos=None):
        for b in range(self.batch):
            e, n = int(entry0[b]), int(n_rows[b])
            pos[b, :, e:e + n] = torch.arange(int(pos0[b]), int(pos0[b]) + n, dtype=torch.int32)

    def evict_rows(self, layer, n, budget, out_table, mass, pos=None, sink=0, recent=0, mass_out=None, pos_out=None):
        if self.fail:
            raise RuntimeError("no memory for the kept indices")
        kept = torch.full((self.batch, self.n_heads, out_table.shape[1] * self.block_size), -1, dtype=torch.int32)
        mass_out.zero_()
        pos_out.fill_(-1)
        for b in range(self.batch):
            for h in range(self.n_heads):
                ks = ref.evict(mass[b, h].numpy(), int(n[b]), int(budget[b]), sink, recent)
                kept[b, h, :len(ks)] = torch.from_numpy(ks)
                mass_out[b, h, :len(ks)] = mass[b, h, ks]
                pos_out[b, h, :len(ks)] = pos[b, h, ks]
        return kept, mass_out, pos_out


def put(c, layer, pos, n):
    x = np.zeros((n, 2, 64), np.float32)
    c.append(layer, x, x, np.arange(pos, pos + n))


def state(c):
    return copy.deepcopy([c.counts, c.block_tables, sorted(c.pool._free), c._floor, c.next_pos])


def test_rollback_refuses_layers_that_were_evicted_apart():
    """80 positions, layer 1 pruned to 8: entry 70 is position 70 in layer 0 and not
    there in layer 1, whose last entries go up to position 79."""
    c = HostCache()
    put(c, 0, 0, 80)
    put(c, 1, 0, 80)
    c.evict(8, sink=0, recent=4, layers=[1])
    before = state(c)
    for n in (1, 5, 7, 8, 70, 79):
        with pytest.raises(ValueError):
            c.truncate(n)
        assert state(c) == before
    c.truncate(80)
    assert state(c) == before
    c.evict(8, sink=0, recent=4)               # now alike: the last 4 entries are 76..79 everywhere
    assert c.counts == [[8, 8]] and c.next_pos == [80]
    c.truncate(5)
    assert c.counts == [[5, 5]] and c.next_pos == [77]
    assert all((c.positions(L)[:, 4] == 76).all() for L in (0, 1))
    for L in (0, 1):
        put(c, L, 77, 2)
        assert (c.positions(L)[:, 4:] == [76, 77, 78]).all()
    assert c.next_pos == [79]
    c.truncate(0)
    assert c.counts == [[0, 0]] and c.next_pos == [0] and c.blocks_in_use == 0
    c.pool.check_invariants()


def test_rollback_of_a_half_appended_step():
    """Without an eviction an entry is a position in every layer, whatever their lengths."""
    c = HostCache(n_layers=3)
    for L in range(3):
        put(c, L, 0, 20)
    put(c, 0, 20, 1)
    put(c, 1, 20, 1)
    c.truncate(20)
    assert c.counts == [[20, 20, 20]] and c.next_pos == [20]
    for n in (-3, -1):
        c.truncate(n)                          # nothing below an empty cache
        assert c.counts == [[0, 0, 0]] and c.next_pos == [0]
    c.pool.check_invariants()


def test_rollback_of_a_batch_is_all_or_nothing():
    """Sequence 1 was pruned to 40 entries, of which it can give back the last 4;
    sequence 0, too short to be pruned, could go back further."""
    c = HostCache(batch=2)
    for L in (0, 1):
        put(c, L, 0, 38)
        c._ensure_layer(1, L, 80)
    for L in (0, 1):
        c.counts[1][L] = 80
    c.next_pos[1] = 80
    c.evict(40, sink=0, recent=4)
    assert c.counts == [[38, 38], [40, 40]]
    before = state(c)
    with pytest.raises(ValueError):
        c.truncate(30)
    assert state(c) == before
    c.truncate(37)
    assert c.counts == [[37, 37], [37, 37]] and c.next_pos == [37, 77]
    c.pool.check_invariants()


def test_appends_continue_the_layer_s_positions():
    c = HostCache()
    for start in (1, 5):
        with pytest.raises(ValueError):
            put(c, 0, start, 3)
    for L in (0, 1):
        put(c, L, 0, 80)
    c.evict(8, sink=0, recent=4)
    for start in (8, 10, 79, 81):              # positions the cache has seen, or a gap
        with pytest.raises(ValueError):
            put(c, 0, start, 2)
    put(c, 0, 80, 2)
    with pytest.raises(ValueError):
        put(c, 1, 82, 1)                       # layer 1 goes on at 80 whatever layer 0 holds
    put(c, 1, 80, 2)
    assert c.next_pos == [82] and c.counts == [[10, 10]]
    assert (c.positions(1)[:, -3:] == [79, 80, 81]).all()


def test_a_failed_eviction_returns_its_blocks():
    c = HostCache(batch=2)
    for L in (0, 1):
        put(c, L, 0, 80)
    before = state(c)
    c.fail = True
    with pytest.raises(RuntimeError):
        c.evict(40, sink=0, recent=4)
    assert state(c) == before
    c.pool.check_invariants()
    c.fail = False
    c.evict(40, sink=0, recent=4)
    assert c.counts[0] == [40, 40] and c.blocks_in_use == 6
    small = HostCache(n_blocks=10)
    for L in (0, 1):
        put(small, L, 0, 80)
    before = state(small)
    with pytest.raises(BlockPoolExhausted):
        small.evict(40, sink=0, recent=4)
    assert state(small) == before


def test_scratch_of_refused_calls_has_no_size():
    """Split lengths that the call refuses ask for no scratch (one of 1 would mean a split an entry)."""
    from draftkv import _lib
    size = _lib.load(require_device=False).dkv_q8_attn_work_bytes
    dims = _lib.DimsS(1, 2, 64, 1)
    assert [size(dims, 4, 1, 1 << 20, s, 0) for s in (1, 100, 129)] == [0, 0, 0]
    assert size(dims, 4, 1, 1 << 20, 128, 0) > size(dims, 4, 1, 1 << 20, 1024, 0) > 65536
