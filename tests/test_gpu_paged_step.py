"""A model on the paged cache (engine.PagedBatch): prompts in chunks, decoding, and speculative decoding, with the tokens
and logits of the engine's own decode plan."""
import numpy as np
import pytest

from llamatov_amd import engine as dr
from llamatov_amd import model as M
from llamatov_amd._lib import LT_KV_F16, LT_KV_F32

pytestmark = pytest.mark.gpu


def case(msg):
    print(f"[gpu-case] {msg}", flush=True)


@pytest.fixture(scope="module")
def tiny(gpu):
    cfg = M.TINY
    m = dr.ResidentModel(cfg, M.synth_weights(cfg, seed=99))
    prompts = [M.random_prompt(cfg, n, seed=n) for n in (6, 11, 3)]
    yield m, prompts
    m.free()


def greedy(m, prompt, n, kv):
    """n greedy tokens of the decode plan, and the logits that the last prompt token gave."""
    plan = dr.DecodePlan(m, dr.Profile(kv_dtype=kv))
    runner = dr.StepGraph(plan)
    logits = np.array(runner.seed(prompt))
    first = plan.read_token()
    runner.capture()
    toks = [first] + runner.replay_tokens(n - 1)
    runner.free()
    plan.free()
    return toks, logits


@pytest.mark.parametrize("kv", [LT_KV_F16, LT_KV_F32])
def test_speculative_decoding_gives_the_greedy_tokens(gpu, tiny, kv):
    """Drafts that are right up to a place and wrong from there: the tokens are the greedy ones, the counts those of the
    right drafts, and the next chunk overwrites the rows of the rejected ones."""
    m, prompts = tiny
    n = 30
    truth = [greedy(m, p, n + 8, kv) for p in prompts]
    cache = dr.PagedKVCache(m.cfg.n_layers, n_pages=24, page=8, nkv=m.cfg.n_head_kv, hd=m.cfg.head_dim, max_seqs=3,
                            max_pages=8, kv_dtype=kv, dev=gpu)
    pb = dr.PagedBatch(m, cache, max_rows=40)
    case(f"speculative decoding kv {kv}")
    # the prompts in two chunks, the second ending in the first new token
    pb.step([p[:2] for p in prompts])
    pb.advance()
    assert cache.lengths() == [2, 2, 2]
    pb.step([p[2:] for p in prompts])
    last = np.cumsum([len(p) - 2 for p in prompts]) - 1
    logits = pb.logits.to_host()
    for b in range(3):
        # both paths round the same products; they part where an activation's quantum falls to the other side of a half,
        # which moves a logit by a small part of their spread
        assert np.abs(logits[last[b]] - truth[b][1]).max() <= 0.05 * truth[b][1].std()
    pb.advance()
    got = [[int(np.argmax(logits[last[b]]))] for b in range(3)]
    rng = np.random.default_rng(4)
    while min(len(g) for g in got) < n:
        chunks, right = [], []
        for b in range(3):
            at, k = len(got[b]), int(rng.integers(0, 5))
            drafts, good = list(truth[b][0][at:at + k]), int(rng.integers(0, k + 1))
            for i in range(good, k):
                drafts[i] = (drafts[i] + 1 + int(rng.integers(0, 100))) % m.cfg.vocab
            if len(got[b]) >= n:
                chunks.append([])
                right.append(None)
                continue
            chunks.append([got[b][-1]] + drafts)
            right.append(good)
        before = cache.lengths()
        pb.step(chunks)
        new = pb.verify()
        for b in range(3):
            if right[b] is None:
                assert new[b] == []
                continue
            assert len(new[b]) == right[b] + 1
            got[b] += new[b]
        assert cache.lengths() == [x + len(y) for x, y in zip(before, new)]
    for b in range(3):
        k = min(len(got[b]), len(truth[b][0]))
        assert got[b][:k] == truth[b][0][:k]
    assert int(pb.err.to_host()[0]) == 0
    cache.release(1)
    assert cache.lengths()[1] == 0
    pb.free()
    cache.free()


def test_sampled_steps_repeat(gpu, tiny):
    """Plain sampled decoding through verify() (no drafts): the same seeds give the same tokens, another seed others."""
    m, prompts = tiny
    case("sampled decoding on the paged cache")

    def play(seed):
        cache = dr.PagedKVCache(m.cfg.n_layers, 24, 8, m.cfg.n_head_kv, m.cfg.head_dim, 3, 8, LT_KV_F16, gpu)
        pb = dr.PagedBatch(m, cache, max_rows=24)
        for b in range(3):
            pb.set_params(b, 1.2, top_k=200, top_p=0.98, seed=seed + b)
        pb.step([p[:-1] for p in prompts])
        pb.advance()
        toks = [[int(p[-1])] for p in prompts]
        for _ in range(12):
            pb.step([t[-1:] for t in toks])
            for t, new in zip(toks, pb.verify()):
                assert len(new) == 1 and 0 <= new[0] < m.cfg.vocab
                t += new
        pb.free()
        cache.free()
        return toks

    a = play(5)
    assert a == play(5) and a != play(6)


def test_paged_batch_refusals(gpu, tiny):
    m, prompts = tiny
    case("PagedBatch refusals")
    c = m.cfg
    with pytest.raises(ValueError):
        dr.PagedBatch(m, dr.PagedKVCache(c.n_layers + 1, 4, 8, c.n_head_kv, c.head_dim, 1, 4, dev=gpu), 8)
    cache = dr.PagedKVCache(c.n_layers, 4, 8, c.n_head_kv, c.head_dim, 1, 4, dev=gpu)
    with pytest.raises(ValueError):
        dr.PagedBatch(m, cache, 0)
    pb = dr.PagedBatch(m, cache, 8)
    with pytest.raises(ValueError):
        pb.step([[1], [2]])
    with pytest.raises(ValueError):
        pb.step([list(range(9))])
    pb.step([[]])
    assert pb.verify() == [[]]
    cache.set_lengths([30])
    with pytest.raises(ValueError):
        pb.step([[1, 2, 3]])
    assert cache.pages == [[]]
    pb.free()
    cache.free()


def test_paged_batch_counts_a_step_once(gpu, tiny):
    """Rows are counted by one advance() or verify() a step; tokens, sequences and sampling settings are checked before."""
    m, prompts = tiny
    case("PagedBatch calls out of order")
    c = m.cfg
    cache = dr.PagedKVCache(c.n_layers, 4, 8, c.n_head_kv, c.head_dim, 2, 4, dev=gpu)
    pb = dr.PagedBatch(m, cache, 8)
    for call in (pb.advance, pb.verify):
        with pytest.raises(RuntimeError):
            call()
    pb.step([prompts[0][:3], []])
    pb.advance()
    for call in (pb.advance, pb.verify):
        with pytest.raises(RuntimeError):
            call()
    assert cache.lengths() == [3, 0]
    for bad in (-1, c.vocab):
        with pytest.raises(ValueError, match="vocabulary"):
            pb.step([[1, bad], []])
    for b, k in ((-1, 40), (2, 40), (0, 0), (0, 1025)):
        with pytest.raises(ValueError):
            pb.set_params(b, 0.8, top_k=k)
    pb.step([[], prompts[1][:2]])
    with pytest.raises(ValueError, match="numbers"):
        pb.verify(u=dr.DevTensor.zeros((1,), np.float32, gpu))
    got = pb.verify()
    assert got[0] == [] and 1 <= len(got[1]) <= 2 and cache.lengths() == [3, len(got[1])] and pb.error() == 0
    with pytest.raises(RuntimeError):
        pb.verify()
    pb.free()
    cache.free()


def test_paged_batch_verifies_with_a_drafter_after_none(gpu, tiny):
    """The verification's workspace grows with what a step needs."""
    m, prompts = tiny
    case("PagedBatch verification, without and with a drafter's logits")
    c = m.cfg
    cache = dr.PagedKVCache(c.n_layers, 8, 8, c.n_head_kv, c.head_dim, 1, 8, dev=gpu)
    pb = dr.PagedBatch(m, cache, 8)
    pb.step([prompts[0]])
    pb.advance()
    pb.step([[1]])
    assert len(pb.verify()[0]) == 1
    pb.step([[2, 3, 4]])
    logits = pb.logits.to_host()[:3]
    best = logits.argmax(1)
    pb.step([[2, int(best[0]), 4]])              # the first draft is the greedy token
    logits = pb.logits.to_host()[:3]
    draft = np.zeros_like(logits)
    draft[0, best[0]] = 1.0
    draft[1, 4] = 1.0
    got = pb.verify(draft_logits=dr.DevTensor.from_host(draft, gpu))[0]
    second = int(logits[1].argmax())
    assert got == [int(best[0]), second] + ([int(logits[2].argmax())] if second == 4 else [])
    pb.free()
    cache.free()
