"""Forwards over the 8-bit cache where the cache's own rounding has no part in the
comparison: the oracle attends to what the device cache holds, so the suite's
tolerances for models apply (2e-2 of max |logit| in bf16, 1e-3 in fp32), and the
engine's tokens equal a loop of single forwards."""
import numpy as np
import pytest

from draftkv import weights as W
from tests.golden.make_golden import SMALL_MODELS
from tests.test_gpu_q8_model import models, rel

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TOL = {"f32": 1e-3, "bf16": 2e-2}


class DeviceValues:
    """The oracle's cache interface over a device cache that has run the same tokens."""

    def __init__(self, cache):
        self.c, self.n = cache, [0] * cache.n_layers
        self.mass = [np.zeros((cache.n_heads, 0)) for _ in range(cache.n_layers)]

    def append(self, layer, k, v, pos):
        self.n[layer] += k.shape[0]
        self.mass[layer] = np.concatenate([self.mass[layer], np.zeros((self.c.n_heads, k.shape[0]))], 1)

    def read(self, layer):
        x = self.c.read_rows(layer, self.n[layer]).cpu().numpy()
        return x[:, :, 0], x[:, :, 1], np.arange(self.n[layer], dtype=np.int64)

    def note_attention(self, layer, probs):
        self.mass[layer] = self.mass[layer] + probs.sum(0)


@pytest.mark.parametrize("name", list(SMALL_MODELS))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("track", [True, False])
def test_forward_over_the_values_that_the_cache_holds(name, dtype, track):
    """Prompts and single tokens; chunks of whole blocks, so that no value is
    rounded again after a row has attended to it.  Without the mass the 80 tokens
    are one call of more than 64 rows a head."""
    from draftkv import Q8KVCache
    m, om = models(name, dtype)
    cache = Q8KVCache(m.n_layers, m.n_kv_heads, m.d_head, n_blocks=16 * m.n_layers, max_blocks_per_seq=16, track_mass=track)
    dv = DeviceValues(cache)
    toks = W.tokens(100, m.vocab_size, seed=9)
    chunk = 16 * max(1, 64 // m.n_rep // 16) if track else 80
    for c0 in range(0, 80, chunk):
        t = toks[c0:min(80, c0 + chunk)]
        got = m.forward(np.array(t), cache, c0)
        want = om.forward(np.array(t), dv, c0)
        assert rel(got, want) < TOL[dtype], (c0, rel(got, want))
    for i in range(80, 83):
        got = m.forward(np.array([toks[i]]), cache, i)
        before = dv.n[0]
        want = om.forward(np.array([toks[i]]), dv, i)
        assert dv.n[0] == before + 1 and rel(got, want) < TOL[dtype], (i, rel(got, want))
    if track:
        for L in range(m.n_layers):
            got = cache.mass[L][0, :, :83].cpu().numpy()
            assert np.abs(got - dv.mass[L]).max() < TOL[dtype] * dv.mass[L].max()


def small_llama():
    from draftkv import LlamaLike
    cfg = W.llama_config(2, 256, 4, 2, 384, 211, head_dim=128, tied=True, dtype="bf16")
    return LlamaLike(W.make_weights(cfg, seed=5, std=0.09, attn_gain=3.0, attn_sharpness=3.0), cfg), cfg["vocab_size"]


def make_cache(m, **kw):
    from draftkv import Q8KVCache
    return Q8KVCache(m.n_layers, m.n_kv_heads, m.d_head, block_size=32, n_blocks=220, max_blocks_per_seq=100, **kw)


@pytest.mark.parametrize("n", [2, 40, 1500])
@pytest.mark.parametrize("track", [True, False])
def test_engine_tokens_equal_a_loop_of_forwards(n, track):
    """The same prompt pass (generate_baseline of no tokens), then greedy single-token forwards."""
    from draftkv import DraftKVEngine
    m, vocab = small_llama()
    prompt = W.tokens(n, vocab, seed=n)
    got = DraftKVEngine(m, seed=0, full_cache_factory=lambda: make_cache(m, track_mass=track)).generate_baseline(prompt, 12, 0.0)
    cache = make_cache(m, track_mass=track)
    DraftKVEngine(m, seed=0, full_cache_factory=lambda: cache).generate_baseline(prompt, 0, 0.0)
    assert cache.length == n - 1
    tok = prompt[-1]
    for i in range(12):
        tok = int(m.forward(np.array([tok]), cache, n - 1 + i)[-1].argmax())
        assert tok == got[n + i], i


def test_engine_starts_over_in_a_cache_that_was_used():
    """The factory returns one cache again and again, pruned in between: every run
    writes it from entry 0, and it goes on at the run's end."""
    from draftkv import DraftKVEngine
    m, vocab = small_llama()
    prompt = W.tokens(90, vocab, seed=3)
    cache = make_cache(m, track_mass=True)
    eng = DraftKVEngine(m, seed=0, full_cache_factory=lambda: cache)
    first = eng.generate_baseline(prompt, 10, 0.0)
    assert cache.length == 99 and cache.next_pos == [99]
    mass = cache.mass[0][:, :, :99].clone()
    cache.evict(40, sink=2, recent=8)
    assert cache.length == 40 and cache.next_pos == [99]
    assert eng.generate_baseline(prompt, 10, 0.0) == first
    assert cache.length == 99 and cache.next_pos == [99]
    assert torch.equal(cache.mass[0][:, :, :99], mass)
    assert (cache.positions(1) == np.arange(99)).all()
    cache.truncate(50)                            # nothing was evicted in this run
    m.forward(np.array([1]), cache, 50)
    cache.pool.check_invariants()


def test_bounded_decoding_in_the_pool_it_needs():
    """A loop that prunes at 64 entries to 32 runs in the blocks of 64 entries a
    layer and one layer's 32 kept ones; one block less is refused."""
    from draftkv import BlockPoolExhausted, Q8KVCache
    m, vocab = small_llama()
    prompt = W.tokens(50, vocab, seed=2)

    def run(n_blocks):
        cache = Q8KVCache(m.n_layers, m.n_kv_heads, m.d_head, block_size=16, n_blocks=n_blocks, max_blocks_per_seq=4,
                          track_mass=True)
        logits = m.forward(np.array(prompt), cache, 0)
        for _ in range(100):
            token = int(logits[-1].argmax())
            if cache.length >= 64:
                cache.evict(32, sink=4, recent=8)
            logits = m.forward(np.array([token]), cache, cache.next_pos[0])
        return cache

    cache = run(m.n_layers * 4 + 2)
    assert cache.next_pos == [150] and 32 <= cache.length <= 64
    assert (cache.positions(0)[:, -8:] == np.arange(142, 150)).all() and (cache.positions(1)[:, :4] == np.arange(4)).all()
    cache.pool.check_invariants()
    with pytest.raises(BlockPoolExhausted):
        run(m.n_layers * 4 + 1)


def test_batches_add_up_the_mass_of_their_own_sequences():
    """Two sequences decoded together with the mass, against each alone (key splits,
    and so the last bits, depend on the batch)."""
    from draftkv import DraftKVEngine, Q8KVCache
    m, vocab = small_llama()
    prompts = [W.tokens(70, vocab, seed=s) for s in (5, 6)]

    def run(ps):
        cache = Q8KVCache(m.n_layers, m.n_kv_heads, m.d_head, block_size=32, n_blocks=30, batch=len(ps),
                          max_blocks_per_seq=5, track_mass=True)
        toks = DraftKVEngine(m, seed=0, full_cache_factory=lambda: cache).generate_baseline_batch(ps, 0, 0.0)
        return toks, [x[:, :, :70].cpu().numpy() for x in cache.mass[:m.n_layers]]

    both, mass = run(prompts)
    for b, p in enumerate(prompts):
        one, alone = run([p])
        assert both[b] == one[0]
        for L in range(m.n_layers):
            assert np.abs(mass[L][b] - alone[L][0]).max() < TOL["bf16"] * alone[L].max()
            assert np.abs(mass[L][b].sum() - m.n_rep * m.n_kv_heads * 69) < 1e-3 * 69     # 69 tokens, weights of sum 1
