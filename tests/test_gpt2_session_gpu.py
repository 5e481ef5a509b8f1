"""A GPT-2 session on the B200: prompts, single tokens and further stretches through the paged caches give the
logits of the oracle's full forward of the same tokens, per element within the bound of
tests/test_gpt2_gpu.py (8 times the rounding noise of bf16 storage plus 1e-2 of the value; the bf16 cache holds the
in-projection's own values)."""
import numpy as np
import pytest

import oracle as O
from _helpers import bf16_bits_to_f32
from test_gpt2_gpu import oracle_forward, storage_sigma, within

pytestmark = pytest.mark.gpu

DIMS = dict(n_layer=2, d_model=128, n_head=2, d_ff=512, vocab=1001, n_ctx=256)


@pytest.fixture(scope="module")
def setup():
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.gpt2 import GPT2, GPT2Config, random_weights
    from tensor_cuda.runtime import Device
    be = CudaBackend(Device.shared(0))
    cfg = GPT2Config(**DIMS)
    w = random_weights(cfg, seed=5, std=0.05)
    return be, cfg, w, GPT2(be, cfg, w)


def read(be, t):
    h = be.read_sync(t)
    return bf16_bits_to_f32(h.data).reshape(h.shape)


def check(cfg, w, ids, lengths, got):
    """Logits after ids[b, :lengths[b]] against the oracle's forward of the whole rows (causal: what follows
    does not matter)."""
    want = oracle_forward(cfg, w, ids)
    sigma = storage_sigma(cfg, w, ids, want)
    at = np.asarray(lengths) - 1
    ok, worst = within(got, want[np.arange(len(ids)), at], sigma)
    assert ok, (worst, sigma)


@pytest.mark.parametrize("page_size", [16, 5])
def test_steps_match_the_full_forward(setup, page_size):
    """A ragged prompt, single tokens, a further ragged stretch, a single token again."""
    be, cfg, w, model = setup
    B = 3
    ids = O.randint_i32(B * 120, 9, cfg.vocab).reshape(B, 120)
    s = model.session(B, page_size=page_size)
    done = [0] * B
    for counts in ([50, 1, 33], [1, 1, 1], [1, 1, 1], [20, 3, 7], [1, 1, 1], [9, 40, 1]):
        n = max(counts)
        step = np.zeros((B, n), np.int32)
        for b, c in enumerate(counts):
            step[b, :c] = ids[b, done[b]:done[b] + c]
        logits = s.step(step, counts)
        done = [d + c for d, c in zip(done, counts)]
        check(cfg, w, ids, done, read(be, logits))
    assert s.lengths == done
    s.release(1)
    assert s.lengths[1] == 0
    s.dispose()


def test_first_step_of_one_token(setup):
    be, cfg, w, model = setup
    ids = O.randint_i32(2, 4, cfg.vocab).reshape(2, 1)
    s = model.session(2)
    check(cfg, w, ids, [1, 1], read(be, s.step(ids)))
    s.dispose()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_generate(setup, cache):
    """Greedy tokens are the steps' largest logits; draws repeat with the same numbers and stay within top_k = 1
    where that is asked; a session goes on where it stopped."""
    be, cfg, w, model = setup
    prompts = [[1, 2, 3, 4, 5], [7], list(range(100, 140))]
    s = model.session(3, cache_dtype=cache)
    greedy = s.generate(prompts, 12, temperature=0.0)
    assert s.lengths == [len(p) + 11 for p in prompts]
    s.dispose()
    t = model.session(3, cache_dtype=cache)
    ids = np.zeros((3, 40), np.int32)
    for row, p in zip(ids, prompts):
        row[:len(p)] = p
    logits = read(be, t.step(ids, [len(p) for p in prompts]))
    for i in range(12):
        best = logits.argmax(1)
        assert best.tolist() == [g[i] for g in greedy]
        logits = read(be, t.step(best.reshape(3, 1).astype(np.int32)))
    t.dispose()
    u = np.random.default_rng(0).random((3, 12))
    draws = []
    for kw in (dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01),) * 2 + (dict(temperature=5.0, top_k=1),):
        s = model.session(3, cache_dtype=cache)
        draws.append(s.generate(prompts, 12, u, **kw))
        s.dispose()
    assert draws[0] == draws[1] and draws[2] == greedy
    assert all(0 <= x < cfg.vocab for row in draws[0] for x in row)


def test_pages_run_out_without_a_trace(setup):
    be, cfg, w, model = setup
    ids = O.randint_i32(2 * 40, 9, cfg.vocab).reshape(2, 40)
    s = model.session(2, n_pages=5, page_size=16)
    s.step(ids[:, :20])
    with pytest.raises(MemoryError, match="free"):
        s.step(ids[:, 20:40])
    assert s.lengths == [20, 20] and s.table.free_pages == 1
    check(cfg, w, ids, [21, 21], read(be, s.step(ids[:, 20:21])))
    with pytest.raises(ValueError, match="context"):
        s.step(np.zeros((2, 250), np.int32))
    with pytest.raises(ValueError, match="counts"):
        s.step(ids[:, :4], [0, 4])
    s.dispose()


def test_sessions_refuse(setup):
    be, cfg, w, model = setup
    with pytest.raises(TypeError, match="cache of f16"):
        model.session(2, cache_dtype="f16")
    s = model.session(1)
    with pytest.raises(ValueError, match="uniform numbers"):
        s.generate([[1, 2]], 3)
    with pytest.raises(ValueError, match="prompts"):
        s.generate([[]], 3, temperature=0.0)
    with pytest.raises(ValueError, match="ids"):
        s.step(np.zeros((2, 3), np.int32))
    s.dispose()


def test_generate_takes_all_or_nothing(setup):
    """A stretch that the pool or the context cannot hold to its end changes nothing; the longest that fits runs."""
    be, cfg, w, model = setup
    s = model.session(2, n_pages=4, page_size=16)
    with pytest.raises(MemoryError, match="free"):
        s.generate([[1, 2, 3], [4]], 31, temperature=0.0)  # 33 and 31 tokens: 3 + 2 pages
    assert s.lengths == [0, 0] and s.table.free_pages == 4
    got = s.generate([[1, 2, 3], [4]], 30, temperature=0.0)  # 32 and 30
    assert s.lengths == [32, 30] and [len(g) for g in got] == [30, 30] and s.table.free_pages == 0
    s.dispose()
    s = model.session(1)
    with pytest.raises(ValueError, match="context"):
        s.generate([[1] * 200], 58, temperature=0.0)  # 257 of 256
    assert s.lengths == [0]
    assert len(s.generate([[1] * 200], 57, temperature=0.0)[0]) == 57 and s.lengths == [256]
    s.dispose()


def test_generate_refuses_settings_before_it_steps(setup):
    """Settings that sample would refuse are refused while nothing has changed."""
    from tensor_cuda.backend import host
    be, cfg, w, model = setup
    s = model.session(2)
    free = s.table.free_pages
    u = np.full((2, 3), 0.5)
    wrong = be.from_host_sync(host("f32", (3,), np.ones(3, np.float32)))
    whole = be.from_host_sync(host("i32", (2,), np.ones(2, np.int32)))
    for kw in (dict(temperature=wrong), dict(top_k=wrong), dict(top_p=whole), dict(min_p=wrong), dict(temperature=None),
               dict(top_p="0.9"), dict(top_k=[1, 2])):
        with pytest.raises((TypeError, ValueError)):
            s.generate([[1, 2, 3], [4]], 3, u, **kw)
        assert s.lengths == [0, 0] and s.table.free_pages == free
    gone = be.from_host_sync(host("f32", (2,), np.ones(2, np.float32)))
    be.dispose(gone)
    with pytest.raises(RuntimeError, match="dispose"):
        s.generate([[1, 2, 3], [4]], 3, u, top_p=gone)
    assert s.lengths == [0, 0] and s.table.free_pages == free
    a = s.generate([[1, 2, 3], [4]], 3, u, temperature=1.0, top_k=whole)
    assert [len(x) for x in a] == [3, 3] and s.lengths == [5, 3]
    s.dispose()


def test_a_session_inside_a_scope(setup):
    """Steps within be.scope keep the session usable behind it; the logits returned are the caller's."""
    be, cfg, w, model = setup
    ids = O.randint_i32(2 * 30, 9, cfg.vocab).reshape(2, 30)
    s = model.session(2)
    first = be.scope(lambda: s.step(ids[:, :20]))
    check(cfg, w, ids, [20, 20], read(be, first))
    check(cfg, w, ids, [21, 21], read(be, s.step(ids[:, 20:21])))
    check(cfg, w, ids, [24, 24], read(be, be.scope(lambda: s.step(ids[:, 21:24]))))
    check(cfg, w, ids, [25, 25], read(be, s.step(ids[:, 24:25])))
    s.dispose()
