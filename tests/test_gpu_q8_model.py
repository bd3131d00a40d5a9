"""Models over the 8-bit cache: forwards, decoding and eviction against the
numpy oracle running over a 64-bit restatement of that cache.

Tolerances, of max |logit|.  fp32 models: 2e-2, since a value of K or V that
fp32 noise moves across a rounding boundary lands on the neighbouring code, up
to 2^-3 of it.  bf16 models: K and V reach the cache off by up to 2^-9 and the
values before them likewise, 2^-8 in all; codes lie 2^-4 to 2^-3 apart, so up to
1/16 of the values land on a neighbour, an rms of (1/16)^(1/2) 2^-3 = 2^-5 where
a bf16 cache has 2^-9: 16 times the suite's bf16 tolerance of 2e-2."""
import numpy as np
import pytest

import oracle
from draftkv import weights as W
from tests import q8_reference as ref
from tests.golden.make_golden import SMALL_MODELS, small_model_cfg, small_model_weights

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TOL = {"f32": 2e-2, "bf16": 16 * 2e-2}


class RefModelCache:
    """One sequence's 8-bit cache behind the oracle's cache interface, with the
    attention mass per KV head and eviction."""

    def __init__(self, n_layers, kv, d, page, pages):
        codes = np.zeros((n_layers * pages, kv, 2, page * d), np.uint8)
        table = np.arange(n_layers * pages).reshape(1, n_layers, pages)
        self.r = ref.RefCache(codes, np.ones((n_layers * pages, kv, 2)), table, page, d)
        self.n, self.kv, self.page, self.pages = [0] * n_layers, kv, page, pages
        self.mass = [np.zeros((kv, 0)) for _ in range(n_layers)]
        self.where = [np.zeros((0,), np.int64) for _ in range(n_layers)]

    def append(self, layer, k, v, pos):
        self.r.append(layer, k[None], v[None], [self.n[layer]], [k.shape[0]])
        self.n[layer] += k.shape[0]
        self.mass[layer] = np.concatenate([self.mass[layer], np.zeros((self.kv, k.shape[0]))], 1)
        self.where[layer] = np.concatenate([self.where[layer], pos])

    def read(self, layer):
        kv = [self.r.entries(0, layer, h, self.n[layer]) for h in range(self.kv)]
        return (np.stack([x[0] for x in kv], 1).astype(np.float32), np.stack([x[1] for x in kv], 1).astype(np.float32),
                self.where[layer])

    def note_attention(self, layer, probs):
        self.mass[layer] = self.mass[layer] + probs.sum(0)

    def evict(self, layer, kept):
        """Keeps the given entries [kv, m], written as an append to empty pages would."""
        m = kept.shape[1]
        rows = [self.r.entries(0, layer, h, self.n[layer]) for h in range(self.kv)]
        for h in range(self.kv):
            for p in range(-(-m // self.page)):
                pid = self.r.table[0, layer, p]
                for i in (0, 1):
                    self.r._put(pid, h, i, 0, rows[h][i][kept[h, p * self.page:(p + 1) * self.page]])
        self.mass[layer] = np.stack([self.mass[layer][h, kept[h]] for h in range(self.kv)])
        self.n[layer] = m
        self.where[layer] = np.full((m,), -1, np.int64)          # before every later token


def models(name, dtype):
    from draftkv import from_config
    cfg = dict(small_model_cfg(W, name))
    wts = small_model_weights(W, name)
    if dtype == "bf16":
        wts = {k: W.round_bf16(v) for k, v in wts.items()}
    cfg["dtype"] = dtype
    return from_config(wts, cfg), oracle.OracleModel(wts, small_model_cfg(W, name))


def rel(got, want):
    return float(np.abs(got.cpu().numpy() - want).max() / np.abs(want).max())


@pytest.mark.parametrize("name", list(SMALL_MODELS))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
def test_forward_decode_and_evict(name, dtype, page):
    from draftkv import Q8KVCache
    m, om = models(name, dtype)
    cache = Q8KVCache(m.n_layers, m.n_kv_heads, m.d_head, block_size=page, n_blocks=40, max_blocks_per_seq=256 // page,
                      track_mass=True)
    rc = RefModelCache(m.n_layers, m.n_kv_heads, m.d_head, page, 256 // page)
    toks = W.tokens(130, m.vocab_size, seed=4)
    chunk = 64 // m.n_rep
    pos = 0

    def run(t):
        nonlocal pos
        got = m.forward(np.array(t), cache, pos)
        want = np.concatenate([om.forward(np.array(t[i:i + chunk]), rc, pos + i) for i in range(0, len(t), chunk)])
        pos += len(t)
        assert rel(got, want) < TOL[dtype], (pos, rel(got, want))

    run(toks[:70])
    for t in toks[70:80]:
        run([t])
    run(toks[80:86])
    for L in range(m.n_layers):
        got = cache.mass[L][0, :, :cache.length].cpu().numpy()
        # weights under scores that differ as the logits may
        assert np.abs(got - rc.mass[L]).max() < TOL[dtype] * rc.mass[L].max()
    kept = cache.evict(40, sink=2, recent=8)
    assert sorted(kept) == list(range(m.n_layers)) and cache.length == 40 and cache.next_pos[0] == 86
    for L in range(m.n_layers):
        rc.evict(L, kept[L][0, :, :40].cpu().numpy())
        assert np.array_equal(cache.positions(L), kept[L][0, :, :40].cpu().numpy())
    for t in toks[86:100]:
        run([t])
    run(toks[100:104])
    # roll back three tokens and go on
    cache.truncate(cache.length - 3)
    assert cache.next_pos[0] == 101
    pos = 101
    for L in range(m.n_layers):
        rc.n[L] -= 3
        rc.mass[L], rc.where[L] = rc.mass[L][:, :-3], rc.where[L][:-3]
    run(toks[110:112])
    with pytest.raises(ValueError):
        m.forward(np.array([1]), cache, 5)
    cache.pool.check_invariants()


def test_prompt_forward_and_greedy_decode_through_the_engine():
    """generate_baseline over an 8-bit cache: the stream equals a greedy loop of
    model.forward over the same kind of cache; long prompts take the prompt kernel."""
    from draftkv import DraftKVEngine, LlamaLike, Q8KVCache
    cfg = W.llama_config(2, 256, 4, 2, 384, 211, head_dim=128, tied=True, dtype="bf16")
    m = LlamaLike(W.make_weights(cfg, seed=5, std=0.09, attn_gain=3.0, attn_sharpness=3.0), cfg)

    def make(batch=1):
        return Q8KVCache(m.n_layers, m.n_kv_heads, m.d_head, block_size=32, n_blocks=200 * batch, batch=batch,
                         max_blocks_per_seq=100)

    for n in (40, 1500):
        prompt = W.tokens(n, cfg["vocab_size"], seed=n)
        eng = DraftKVEngine(m, seed=0, full_cache_factory=make)
        got = eng.generate_baseline(prompt, 12, 0.0)
        assert len(got) == n + 12 and got[:n] == list(prompt)
        # teacher-forced: each emitted token is the argmax of its row, up to near ties
        cache = make()
        lg = m.forward(np.array(got[:-1]), cache, 0)[n - 1:].float()
        top = lg.max(-1).values
        mine = lg[torch.arange(12), torch.tensor(got[n:]).to(lg.device)]
        assert ((top - mine) <= TOL["bf16"] * lg.abs().max()).all()
    two = [W.tokens(30, cfg["vocab_size"], seed=s) for s in (1, 2)]
    eng = DraftKVEngine(m, seed=0, full_cache_factory=lambda: make(2))
    both = eng.generate_baseline_batch(two, 8, 0.0)
    for p, row in zip(two, both):
        assert row == DraftKVEngine(m, seed=0, full_cache_factory=make).generate_baseline(p, 8, 0.0)
    with pytest.raises(NotImplementedError):
        DraftKVEngine(m, seed=0, full_cache_factory=make).generate(two[0], 8, 0.0)


def test_forward_refuses_what_does_not_fit():
    from draftkv import DraftKVError, LlamaLike, Q8KVCache
    cfg = W.llama_config(2, 128, 4, 2, 192, 101, head_dim=64, tied=True, dtype="f32")
    m = LlamaLike(W.make_weights(cfg, seed=5, std=0.09), cfg)
    with pytest.raises(TypeError):
        m.forward(np.array([1]), Q8KVCache(2, 2, 128, n_blocks=8, max_blocks_per_seq=4), 0)
    with pytest.raises(TypeError):
        m.forward(np.array([1]), Q8KVCache(3, 2, 64, n_blocks=8, max_blocks_per_seq=4), 0)
    cache = Q8KVCache(2, 2, 64, n_blocks=8, max_blocks_per_seq=4, track_mass=True)
    ext = Q8KVCache.from_storage(cache.codes, cache.scale, cache.table_dev)
    with pytest.raises(TypeError):
        m.forward(np.array([1]), ext, 0)
    m.forward(np.array([1, 2, 3]), cache, 0)
    with pytest.raises(ValueError):
        m.forward(np.array([1]), cache, 7)
    # 33 tokens x 2 heads a KV head are more rows than the mass takes in one launch
    w = m.work(1, 40, cache.capacity_tokens, 0, cache)
    cache.ensure(0, 40)
    p0 = torch.tensor([3], dtype=torch.int32, device="cuda")
    tok = torch.zeros(33, dtype=torch.int32, device="cuda")
    with pytest.raises(DraftKVError):
        m.forward_raw(cache, None, tok.data_ptr(), 33, p0, 1, 33, None, w, 40, cache.capacity_tokens, graph=False)
    with pytest.raises(ValueError):
        Q8KVCache(2, 2, 64, n_blocks=8, max_blocks_per_seq=4).evict(4)
