"""Search with beams through the engine: against a plain search whose logits
come from requests of their own, without forks or shared blocks."""

import math

import pytest
import torch

import fusioninfer_amd.ops as ops
from fusioninfer_amd.config import CacheConfig, EngineConfig, SchedulerConfig
from fusioninfer_amd.engine.block_manager import BlockManager
from fusioninfer_amd.engine.llm_engine import (
    InsufficientBlocksError,
    LLMEngine,
)
from fusioninfer_amd.engine.sequence import SamplingParams, Sequence
from fusioninfer_amd.models.registry import get_model_config
from test_kazozen import make_engine as make_kazozen
from test_kazozen import small_config as kazozen_config
from test_momedra import make_engine as make_momedra
from test_momedra import small_config as momedra_config
from test_pinuvik import make_engine as make_pinuvik
from test_pinuvik import small_config as pinuvik_config
from test_sefalorn import make_engine as make_sefalorn
from test_sefalorn import small_config as sefalorn_config
from test_sufavik import make_engine as make_sufavik
from test_sufavik import small_config as sufavik_config
from test_vatunex import make_engine as make_vatunex
from test_vatunex import small_config as vatunex_config


def make_engine(device="cpu", blocks=128, seqs=16, max_len=256, budget=1024,
                model="tiny-qwen3", layers=None, eager=True, **cache):
    mc = get_model_config(model)
    if layers:
        mc.num_layers = layers
    return LLMEngine(EngineConfig(
        model=mc, cache=CacheConfig(num_gpu_blocks=blocks, **cache),
        scheduler=SchedulerConfig(max_num_seqs=seqs,
                                  max_num_batched_tokens=budget,
                                  max_model_len=max_len),
        enforce_eager=eager, seed=3), device=device)


def logprobs_after(eng, prompt, tokens):
    """log-probabilities after prompt and tokens, by a request of its own that
    decodes the tokens one by one, in 64 bits."""
    out = eng.forced_step([("plain", prompt, [len(prompt) - 1])])
    for t in tokens:
        out = eng.forced_step([("plain", [t], [0])])
    eng.forced_step([], ["plain"])
    return torch.log_softmax(out[0].double().cpu(), dim=0)


def plain_search(eng, prompt, width, steps, stops=(), penalty=1.0):
    """[(tokens, cumulative, score)], best first; every step is run."""
    beams, done, known = [((), 0.0)], [], {}
    for _ in range(steps):
        cands = []
        for i, (toks, c) in enumerate(beams):
            if toks not in known:
                known[toks] = logprobs_after(eng, prompt, toks)
            lp = known[toks]
            first = torch.topk(lp, min(len(lp), width * (1 + len(stops))))
            cands += [(-(c + v), i, t) for v, t in zip(
                first.values.tolist(), first.indices.tolist())]
        old, beams = beams, []
        for s, i, t in sorted(cands):
            if len(beams) == width:
                break
            toks = old[i][0] + (t,)
            if t in stops:
                done.append((toks, -s))
            else:
                beams.append((toks, -s))
    done += beams
    done = [(list(t), c, c / len(t) ** penalty) for t, c in done]
    return sorted(done, key=lambda h: -h[2])[:width]


def agree(got, want):
    """Tokens as they are; cumulative scores are rounded to fp32 at each step,
    and each step's ln S is off by less than 1e-5."""
    assert [h.token_ids for h in got] == [w[0] for w in want]
    for h, w in zip(got, want):
        n = len(w[0])
        assert abs(h.cumulative_logprob - w[1]) <= n * (
            1e-5 + 2.0 ** -24 * abs(w[1]))


def nothing_held(eng):
    assert not eng._forced
    assert eng.block_manager.num_free() == eng.block_manager.num_blocks
    if eng.state_manager is not None:
        assert eng.state_manager.num_free() == eng.state_manager.num_slots


@pytest.mark.parametrize("n", [1, 13, 16, 31])
@pytest.mark.parametrize("width", [1, 3, 5])
def test_search_matches_plain_one(n, width):
    eng = make_engine()
    prompt = [(7 * i + n) % 1024 for i in range(n)]
    got, = eng.beam_search([prompt], width, max_tokens=6)
    assert len(got) == width
    assert all(h.finish_reason == "length" for h in got)
    agree(got, plain_search(eng, prompt, width, 6))
    nothing_held(eng)


def test_searches_side_by_side():
    """Prompts of other lengths in one batch, more than fit at once, in
    portions of a step's budget."""
    eng = make_engine(seqs=7, budget=16)
    prompts = [[(11 * i + n) % 1024 for i in range(n)] for n in (5, 40, 17, 16)]
    got = eng.beam_search(prompts, 3, max_tokens=4)
    for g, p in zip(got, prompts):
        agree(g, plain_search(eng, p, 3, 4))
    nothing_held(eng)


@pytest.mark.parametrize("penalty", [0.0, 1.0, 2.5, -0.5])
def test_stop_tokens(penalty):
    """Tokens that the free search meets at several places end hypotheses."""
    eng = make_engine()
    prompt = [5, 6, 7, 8, 9]
    free, = eng.beam_search([prompt], 3, max_tokens=5)
    stops = {free[0].token_ids[1], free[1].token_ids[3], 1000}
    got, = eng.beam_search([prompt], 3, max_tokens=5, stop_token_ids=stops,
                           length_penalty=penalty)
    want = plain_search(eng, prompt, 3, 5, stops, penalty)
    agree(got, want)
    for h, w in zip(got, want):
        ended = h.token_ids[-1] in stops
        assert h.finish_reason == ("stop" if ended else "length")
        assert abs(h.score - w[2]) <= 1e-4 * max(1, abs(w[2]))
    nothing_held(eng)


def test_ends_at_the_longest_sequence():
    eng = make_engine(max_len=32)
    got, = eng.beam_search([[3] * 28], 2, max_tokens=50)
    assert [len(h.token_ids) for h in got] == [4, 4]
    nothing_held(eng)


FAMILIES = [
    (make_vatunex, vatunex_config), (make_pinuvik, pinuvik_config),
    (make_momedra, momedra_config), (make_sefalorn, sefalorn_config),
    (make_sufavik, sufavik_config), (make_kazozen, kazozen_config)]


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("family", range(len(FAMILIES)))
def test_models_with_states(family, device):
    make, config = FAMILIES[family]
    eng, _ = make(config(), device, max_seqs=4)
    prompt = [(5 * i + 1) % 60 for i in range(18)]
    got, = eng.beam_search([prompt], 3, max_tokens=5)
    agree(got, plain_search(eng, prompt, 3, 5))
    with pytest.raises(ValueError):
        eng.beam_search([prompt], 5)     # four slots
    nothing_held(eng)


def test_blocks_run_out():
    eng = make_engine(blocks=4)
    with pytest.raises(InsufficientBlocksError):
        eng.beam_search([[1] * 30], 4, max_tokens=20)
    nothing_held(eng)
    got, = eng.beam_search([[1] * 30], 2, max_tokens=2)
    assert len(got) == 2
    nothing_held(eng)


def test_fewer_searches_at_once_where_blocks_run_out(monkeypatch):
    """Seats for eight searches, blocks for two of them."""
    from fusioninfer_amd.engine import beam_search as module

    tried, run = [], module.BeamSearcher.run
    monkeypatch.setattr(module.BeamSearcher, "run", lambda self, prompts: (
        tried.append(len(prompts)), run(self, prompts))[1])
    eng = make_engine(blocks=8)
    prompts = [[(9 * i + n) % 1024 for i in range(30)] for n in range(5)]
    got = eng.beam_search(prompts, 2, max_tokens=2)
    assert tried[0] == 5 and sum(tried[-3:]) == 5
    for g, p in zip(got, prompts):
        agree(g, plain_search(eng, p, 2, 2))
    nothing_held(eng)


def test_served_requests_stay_as_they_are():
    """A search between the steps of requests that are served."""
    prompts = [[9, 8, 7] * 7, [4] * 30]
    alone = [o.output_token_ids for o in make_engine().generate(
        prompts, SamplingParams(max_tokens=8))]
    eng = make_engine()
    ids = [eng.add_request(p, SamplingParams(max_tokens=8)) for p in prompts]
    done = {}
    for i in range(40):
        for o in eng.step():
            if o.finished:
                done[o.request_id] = o.output_token_ids
        if i == 3:
            eng.beam_search([[2, 3, 4]], 3, max_tokens=3)
        if len(done) == len(ids):
            break
    assert [done[i] for i in ids] == alone
    nothing_held(eng)


def test_refusals():
    eng = make_engine(max_len=64)
    for call in [
        lambda: eng.beam_search([[1]], 0),
        lambda: eng.beam_search([[1]], 17),
        lambda: eng.beam_search([[1]], 2, max_tokens=0),
        lambda: eng.beam_search([[]], 2),
        lambda: eng.beam_search([[1] * 64], 2),
    ]:
        with pytest.raises(ValueError):
            call()
    assert eng.beam_search([], 2) == []
    eng.forced_step([("a", [1, 2], [1])])
    with pytest.raises(ValueError):
        eng.fork_forced("a", "a")
    eng.release_forced(["a", "b"])
    nothing_held(eng)


def test_refuses_more_beams_than_a_choice_takes(monkeypatch):
    """Before the first step: 256 beams of a vocabulary beyond 163840, say."""
    eng = make_engine()
    monkeypatch.setattr(ops, "MOST_CHUNKS", 3)
    with pytest.raises(ValueError):
        eng.beam_search([[1, 2, 3]], 4)
    assert eng.num_prefilled_tokens == 0
    assert len(eng.beam_search([[1, 2, 3]], 3, max_tokens=2)[0]) == 3


@pytest.mark.parametrize("penalty", [float("nan"), float("inf"), 400.0,
                                     -400.0])
def test_refuses_length_penalties_out_of_range(penalty):
    """Lengths to their power would be infinite, or 0."""
    eng = make_engine()
    with pytest.raises(ValueError):
        eng.beam_search([[1, 2, 3]], 2, max_tokens=8, length_penalty=penalty)
    assert eng.num_prefilled_tokens == 0
    for p in (50.0, -50.0):
        got, = eng.beam_search([[1, 2, 3]], 2, max_tokens=8, length_penalty=p)
        assert all(math.isfinite(h.score) for h in got)


def test_fork_of_blocks():
    bm = BlockManager(8, 4)
    a = Sequence("a", [1] * 10, SamplingParams())
    bm.allocate(a)
    b, c = (Sequence(n, [1] * 10, SamplingParams()) for n in "bc")
    src, dst, filled = bm.fork(a, b, 10)
    assert (src, filled) == (a.block_ids[2], 2) and dst not in a.block_ids
    assert b.block_ids == a.block_ids[:2] + [dst]
    assert bm.fork(a, c, 8) is None and c.block_ids == a.block_ids[:2]
    assert bm.num_free() == 4
    bm.free(a)
    assert bm.num_free() == 5        # only the partly filled one
    bm.free(b)
    bm.free(c)
    assert bm.num_free() == 8 and not bm.ref_count


def test_logprobs_of_many_tokens_and_few():
    """Requests that ask for other numbers of them, and for more than one
    launch finds."""
    eng = make_engine()
    prompt = [3, 1, 4] * 5
    few, many = (eng.add_request(prompt, SamplingParams(
        max_tokens=2, logprobs=k)) for k in (2, 400))
    done = {}
    while len(done) < 2:
        for o in eng.step():
            if o.finished:
                done[o.request_id] = o.logprobs
    for (a, some), (b, more) in zip(done[few], done[many]):
        assert math.isclose(a, b, rel_tol=1e-6)
        assert len(some) == 2 and len(more) == 400
        assert list(some) == list(more)[:2]
    assert ops.MOST_CHOICES < 400


# --------------------------------------------------------------------- GPU

@pytest.mark.gpu
@pytest.mark.parametrize("eager", [True, False])
@pytest.mark.parametrize("cache", ["auto", "fp8"])
def test_gpu_scores_are_those_of_the_tokens(eager, cache):
    """Each hypothesis' score against a request of its own that decodes its
    tokens: other batch sizes round products of bf16 elsewhere, so a
    log-probability (of logits below 8, half a bf16 step 2^-6) may be off by
    a few of those; a wrong page is off by whole ones."""
    eng = make_engine("cuda:0", model="Qwen3-0.6B", layers=4, blocks=256,
                      eager=eager, kv_cache_dtype=cache)
    prompts = [[(7 * i + n) % 5000 for i in range(n)] for n in (5, 45, 128)]
    for prompt, got in zip(prompts, eng.beam_search(prompts, 4,
                                                    max_tokens=20)):
        assert len(got) == 4
        assert len({tuple(h.token_ids) for h in got}) == 4
        for h in got:
            total, out = 0.0, eng.forced_step(
                [("plain", prompt, [len(prompt) - 1])])
            for t in h.token_ids:
                total += torch.log_softmax(out[0].double(), 0)[t].item()
                out = eng.forced_step([("plain", [t], [0])])
            eng.forced_step([], ["plain"])
            assert abs(total - h.cumulative_logprob) <= \
                len(h.token_ids) * 4 * 2.0 ** -6
    nothing_held(eng)


@pytest.mark.gpu
def test_gpu_one_beam_is_greedy():
    eng = make_engine("cuda:0", model="Qwen3-0.6B", layers=4, blocks=256)
    prompt = list(range(20, 70))
    got, = eng.beam_search([prompt], 1, max_tokens=12)
    out = eng.forced_step([("plain", prompt, [len(prompt) - 1])])
    for t in got[0].token_ids:
        assert out[0].argmax().item() == t
        out = eng.forced_step([("plain", [t], [0])])
    eng.forced_step([], ["plain"])


@pytest.mark.gpu
def test_gpu_logprobs_of_requests():
    """Tokens' and prompts' log-probabilities as torch has them."""
    eng = make_engine("cuda:0", model="Qwen3-0.6B", layers=2, blocks=256)
    prompt = list(range(30, 60))
    out, = eng.generate([prompt], SamplingParams(
        max_tokens=3, logprobs=4, prompt_logprobs=2))
    full = prompt + out.output_token_ids[:1]
    logits = eng.forced_step([("plain", prompt, list(range(len(prompt))))])
    eng.forced_step([], ["plain"])
    lp = torch.log_softmax(logits.double(), dim=1)
    assert out.prompt_logprobs[0] is None
    for i in range(1, len(prompt)):
        of, top = out.prompt_logprobs[i]
        # the same step but for the rows that the batch's logits cover
        assert abs(of - lp[i - 1, full[i]].item()) <= 4 * 2.0 ** -6
        assert len(top) == 2 and list(top.values()) == sorted(
            top.values(), reverse=True)
    of, top = out.logprobs[0]
    assert out.output_token_ids[0] in top and len(top) == 4
    assert top[out.output_token_ids[0]] == of == max(top.values())


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("batch", [1, 5])
def test_logprobs_are_those_of_the_logits(device, batch, monkeypatch):
    """What requests are given against torch's log-softmax, in 64 bits, of the
    same logits; decode steps of one row, too."""
    from test_search_ops import HALF, away

    seen, entries_of = [], LLMEngine._logprob_entries

    def entries(self, logits, ks, ids):
        before = logits.double().cpu()
        got = entries_of(self, logits, ks, ids)
        seen.append((before, list(ks), list(ids), got))
        return got

    monkeypatch.setattr(LLMEngine, "_logprob_entries", entries)
    eng = make_engine(device, layers=2, blocks=256, **(
        {} if device == "cpu" else {"model": "Qwen3-0.6B"}))
    prompts = [[(17 * i + n) % 1000 for i in range(20 + n)]
               for n in range(batch)]
    eng.generate(prompts, SamplingParams(max_tokens=3, logprobs=7,
                                         prompt_logprobs=20))
    assert min(len(ks) for _, ks, _, _ in seen) == batch \
        and max(len(ks) for _, ks, _, _ in seen) >= 19
    for logits, ks, ids, got in seen:
        lp = torch.log_softmax(logits, 1)
        off = away(lp.shape[1])
        for row, k, t, (of, top) in zip(lp, ks, ids, got):
            assert abs(of - row[t].item()) <= off - HALF * row[t].item()
            want = row.topk(k).values
            assert len(top) == k
            for v, (i, w) in zip(want.tolist(), top.items()):
                # the i-th, and its own token's
                assert abs(w - v) <= off - HALF * v
                assert abs(w - row[i].item()) <= off - HALF * v
