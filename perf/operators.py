"""What is timed of the operators that a search with beams runs on: the
choice over beams and vocabulary, log-probabilities of top and given tokens,
and copies of cache pages and state slots.

A case is one call. Vocabularies, layers, heads and block sizes are those of
the registry's models (Qwen3-8B, Qwen3-30B-A3B, Llama-3-8B) and of the design
that ``bench.py --mixer-compare`` names Vatunex.
"""

import math

import torch

own = False

DEV = "cuda:0"
INF = float("inf")
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32,
          "fp8": torch.float8_e4m3fn}


# ------------------------------------------------------------------ cases

def _beams(name, groups, beams, vocab, dtype="bf16", pad=0, masked=0.0):
    """groups searches of ``beams`` beams each, twice as many candidates as
    beams; rows of logits are ``pad`` columns apart from one another;
    masked: share of the tokens that a grammar forbids (-inf)."""
    c = {"op": "beam", "groups": groups, "beams": beams, "vocab": vocab,
         "k": 2 * beams, "dtype": dtype, "pad": pad, "masked": masked}
    return dict(c, name=name) if name else c


def _top(name, rows, k, vocab, dtype="bf16", pad=0, masked=0.0, given=True):
    """log-probabilities of the k first tokens of every row and of a given
    one."""
    c = {"op": "top", "rows": rows, "k": k, "vocab": vocab, "dtype": dtype,
         "pad": pad, "masked": masked, "given": given}
    return dict(c, name=name) if name else c


def _pages(name, tensors, heads, width, pairs, dtype="bf16", block=16,
           partly=True):
    """pages [heads, block, width] of every cache tensor, copied whole or as
    far as they are filled."""
    c = {"op": "pages", "tensors": tensors, "heads": heads, "block": block,
         "width": width, "pairs": pairs, "dtype": dtype, "partly": partly}
    return dict(c, name=name) if name else c


def _states(name, layers, width, state, conv, pairs):
    """convolution tail [conv - 1, width] and state [width, state] of every
    recurrent layer, fp32."""
    c = {"op": "states", "layers": layers, "width": width, "state": state,
         "conv": conv, "pairs": pairs}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's request with four beams: every generated token
        _beams("beam_one", 1, 4, 151936),
        # a model with a small vocabulary and fp32 logits, rows cut from
        # wider ones
        _beams("beam_small", 16, 5, 32000, "fp32", pad=67),
        # few wide searches, as for n-best lists
        _beams("beam_wide", 2, 32, 128256),
        # a full batch of searches
        _beams("beam_full", 64, 8, 151936),
        # one request with logprobs: every generated token
        _top("top_one", 1, 20, 151936, "fp32"),
        # decode of a batch whose requests ask for logprobs, under grammars
        _top("top_decode", 61, 5, 151936, "fp32", masked=0.9),
        # the prompt's logprobs, as for choosing among answers
        _top("top_prompt", 1531, 1, 151936),
        # likelihood of given tokens alone, as for perplexity
        _top("top_score", 2048, 0, 152064),
        # one request's beams go apart: three copies of a page partly filled
        _pages("fork_one", 72, 8, 128, 3),
        # a full batch's beams go apart
        _pages("fork_full", 72, 8, 128, 320),
        # pages of an e4m3 cache change place, whole
        _pages("move_fp8", 96, 4, 128, 512, "fp8", partly=False),
        # states of the recurrent layers go with their beams
        _states("fork_states", 8, 4096, 16, 4, 48),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def _vocab(rng):
    return rng.choice([32000, 128256, 151936, 152064, rng.randint(5, 1500),
                       rng.randint(1500, 160000)])


def draw(rng):
    op = rng.choice(["beam", "beam", "top", "top", "pages", "states"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    pad = rng.choice([0, 0, rng.randint(1, 200)])
    masked = rng.choice([0.0, 0.0, rng.uniform(0.05, 0.999)])
    size = 2 if dtype == "bf16" else 4
    if op == "beam":
        vocab, beams = _vocab(rng), _log_int(rng, 1, 32)
        most = max(1, min(64, 150_000_000 // (size * vocab * beams)))
        return _beams(None, _log_int(rng, 1, most), beams, vocab, dtype, pad,
                      masked)
    if op == "top":
        vocab = _vocab(rng)
        most = max(1, min(2048, 600_000_000 // (size * vocab)))
        k = min(vocab, rng.choice([0, 1, rng.randint(2, 20)]))
        return _top(None, _log_int(rng, 1, most), k, vocab, dtype, pad,
                    masked, k == 0 or rng.random() < 0.7)
    if op == "pages":
        tensors, heads = rng.choice([4, 7, 32, 72, 96]), rng.randint(1, 8)
        width, block = rng.choice([64, 96, 128, 288]), rng.choice([16, 16, 32])
        dtype = rng.choice(["bf16", "bf16", "fp8"])
        page = tensors * heads * width * block * (2 if dtype == "bf16" else 1)
        most = max(1, min(512, 400_000_000 // page))
        return _pages(None, tensors, heads, width, _log_int(rng, 1, most),
                      dtype, block, rng.random() < 0.7)
    return _states(None, rng.randint(1, 12), rng.choice([96, 1000, 2048, 4096]),
                   rng.choice([1, 16, 16]), rng.choice([2, 4]),
                   _log_int(rng, 1, 64))


# ---------------------------------------------------------------- prepare

def _logits(case, rows, gen):
    """Rows as a model gives them: a broad bulk, and a few dozen tokens that
    stand out."""
    vocab = case["vocab"]
    x = torch.randn(rows, vocab + case["pad"], generator=gen, device=DEV)
    x *= 2.0
    at = torch.randint(0, vocab, (rows, 32), generator=gen, device=DEV)
    up = torch.rand(rows, 32, generator=gen, device=DEV)
    x.scatter_add_(1, at, 4.0 - 3.0 * torch.log(up.clamp(min=1e-6)))
    if case["masked"]:
        gone = torch.rand(x.shape, generator=gen, device=DEV)
        x.masked_fill_(gone < case["masked"], -INF)
    return x.to(DTYPES[case["dtype"]])[:, :vocab]


def _pairs(gen, pairs, slots):
    at = torch.randperm(slots, generator=gen, device=DEV).to(torch.int32)
    # beams that go on from the same one read the same page
    live = at[torch.randint(0, pairs, (pairs,), generator=gen, device=DEV)]
    return live.contiguous(), at[pairs:2 * pairs].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    if case["op"] == "beam":
        g, b = case["groups"], case["beams"]
        scores = -30.0 * torch.rand(g, 1, generator=gen, device=DEV) \
            - 3.0 * torch.rand(g, b, generator=gen, device=DEV)
        return {"op": "beam", "logits": _logits(case, g * b, gen),
                "scores": scores, "k": case["k"]}
    if case["op"] == "top":
        logits = _logits(case, case["rows"], gen)
        given = torch.randint(0, case["vocab"], (case["rows"],),
                              generator=gen, device=DEV)
        return {"op": "top", "logits": logits, "k": case["k"],
                "given": given if case["given"] else None}
    slots = 2 * case["pairs"] + 5
    src, dst = _pairs(gen, case["pairs"], slots)
    if case["op"] == "pages":
        pool = torch.randn(case["tensors"], slots, case["heads"],
                           case["block"], case["width"], generator=gen,
                           device=DEV, dtype=torch.bfloat16)
        pool = pool.to(DTYPES[case["dtype"]])
        filled = torch.randint(1, case["block"] + 1, (case["pairs"],),
                               generator=gen, device=DEV)
        return {"op": "pages", "pool": pool, "tensors": list(pool),
                "src": src, "dst": dst,
                "tokens": filled.to(torch.int32) if case["partly"] else None}
    tails = torch.randn(case["layers"], slots, case["conv"] - 1,
                        case["width"], generator=gen, device=DEV)
    states = torch.randn(case["layers"], slots, case["width"], case["state"],
                         generator=gen, device=DEV)
    return {"op": "states", "tails": tails, "states": states,
            "tensors": list(tails) + list(states), "src": src, "dst": dst}


# -------------------------------------------------------------------- run

def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "beam":
        return _beam_plain(state["logits"], state["scores"], state["k"])
    if state["op"] == "top":
        return _top_plain(state["logits"], state["k"], state["given"])
    src, dst = state["src"].long(), state["dst"].long()
    if state["op"] == "pages":
        return _pages_plain(state["pool"], src, dst, state["tokens"])
    state["tails"][:, dst] = state["tails"][:, src]
    state["states"][:, dst] = state["states"][:, src]
    return state["tails"], state["states"]


def _run_own(state):
    import fusioninfer_amd.ops as ops

    if state["op"] == "beam":
        return tuple(ops.beam_select(state["logits"], state["scores"],
                                     state["k"]))
    if state["op"] == "top":
        return tuple(ops.top_logprobs(state["logits"], state["k"],
                                      state["given"]))
    ops.copy_blocks_(state["tensors"], state["src"], state["dst"],
                     state.get("tokens"))
    if state["op"] == "pages":
        return state["pool"]
    return state["tails"], state["states"]


def _first_k(x, k):
    """The k largest of every row, equal ones by index: logits and tokens.
    A key of 64 bits holds a logit's order and the index below it."""
    bits = x.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    index = torch.arange(x.shape[1], device=x.device)
    key = (order << 32) + (x.shape[1] - 1 - index)
    token = x.shape[1] - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    return torch.gather(x, 1, token), token


def _log_sum(x):
    """ln sum exp of every row, the sum and its logarithm in 64 bits."""
    m = x.amax(1, keepdim=True)
    return m.double() + torch.exp(x - m).sum(1, keepdim=True,
                                             dtype=torch.float64).log()


def _beam_plain(logits, scores, k):
    x = logits.float()
    groups, beams = scores.shape
    each = min(k, x.shape[1])
    value, token = _first_k(x, each)
    z, c = _log_sum(x), scores.reshape(-1, 1).double()
    alive = torch.isfinite(z) & torch.isfinite(c) & (value > -INF)
    s = torch.where(alive, c + (value.double() - z), -INF)
    s = s.view(groups, beams * each)
    s = torch.nn.functional.pad(s, (0, max(0, k - beams * each)), value=-INF)
    s, at = torch.sort(s, dim=1, descending=True, stable=True)
    s, at = s[:, :k], at[:, :k].clamp(max=beams * each - 1)
    token = torch.gather(token.view(groups, -1), 1, at)
    none = s == -INF
    return (s.float(), torch.where(none, -1, at // each).int(),
            torch.where(none, -1, token).int())


def _top_plain(logits, k, given):
    x = logits.float()
    z = _log_sum(x)
    some = torch.isfinite(z)
    if k:
        value, token = _first_k(x, k)
        first = torch.arange(k, device=x.device).expand_as(token)
        top = torch.where(some, value.double() - z, float("nan")).float()
        token = torch.where(some, token, first).int()
    else:
        top, token = x.new_empty(len(x), 0), some.new_empty(len(x), 0).int()
    if given is None:
        return top, token, None
    at = given.view(-1, 1).long()
    of = torch.gather(x, 1, at.clamp(0, x.shape[1] - 1)).double() - z
    of = torch.where((at >= 0) & (at < x.shape[1]), of, -INF)
    return top, token, torch.where(some, of, float("nan")).float().view(-1)


def _pages_plain(pool, src, dst, tokens):
    # e4m3 pages are moved as the bytes they are
    raw = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    if tokens is None:
        raw[:, dst] = raw[:, src]
        return pool
    row = torch.arange(raw.shape[3], device=raw.device)
    held = (row < tokens.view(-1, 1)).view(1, -1, 1, raw.shape[3], 1)
    raw[:, dst] = torch.where(held, raw[:, src], raw[:, dst])
    return pool


# ------------------------------------------------------------------- work

def work(case):
    if case["op"] in ("beam", "top"):
        size = 2 if case["dtype"] == "bf16" else 4
        if case["op"] == "beam":
            rows = case["groups"] * case["beams"]
            out = 12 * case["groups"] * case["k"] + 4 * rows
        else:
            rows = case["rows"]
            out = 8 * rows * case["k"] + (12 * rows if case["given"] else 0)
        # maximum, difference, exponential and sum of every logit
        return {"bytes": rows * case["vocab"] * size + out,
                "flops": 4 * rows * case["vocab"]}
    if case["op"] == "pages":
        size = 2 if case["dtype"] == "bf16" else 1
        held = (case["block"] + 1) / 2 if case["partly"] else case["block"]
        each = case["tensors"] * case["heads"] * held * case["width"] * size
    else:
        each = 4 * case["layers"] * case["width"] * \
            (case["conv"] - 1 + case["state"])
    return {"bytes": 2 * case["pairs"] * each + 8 * case["pairs"], "flops": 0}


# ------------------------------------------------------------------ exact

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "beam":
        return _beam_exact(state["logits"], state["scores"], state["k"])
    if case["op"] == "top":
        return _top_exact(state["logits"], state["k"], state["given"])
    # copies are of bits
    return None


def _beam_exact(logits, scores, k):
    groups, beams = scores.shape
    out = torch.full((groups, k), -INF, dtype=torch.float64, device=DEV)
    for g in range(groups):
        x = logits[g * beams:(g + 1) * beams].to(torch.float64)
        p = torch.log_softmax(x, dim=1) + scores[g].to(torch.float64)[:, None]
        p = p[torch.isfinite(p)]
        best = torch.sort(p, descending=True).values[:k]
        out[g, :best.numel()] = best
    return out, None, None


def _top_exact(logits, k, given):
    top, of = [], []
    for i in range(0, logits.shape[0], 64):
        p = torch.log_softmax(logits[i:i + 64].to(torch.float64), dim=1)
        if k:
            # any exact value: rows with no distribution are NaN throughout
            top.append(torch.sort(p, dim=1, descending=True).values[:, :k])
        if given is not None:
            of.append(p.gather(1, given[i:i + 64, None]).view(-1))
    first = torch.cat(top) if top else logits.new_zeros(
        logits.shape[0], 0, dtype=torch.float64)
    return first, None, torch.cat(of) if of else None
