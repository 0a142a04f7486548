"""Choice of beams, top log-probabilities and copies of blocks, on the CPU and
on the GPU, against plain implementations in 64 bits."""

import math

import numpy as np
import pytest
import torch

import fusioninfer_amd.ops as ops

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = 2.0 ** -24  # half a step of fp32, relative


def away(V):
    """How far ln S may be off, S = sum exp(l - m). A term exp(t), t = l - m <= 0: t and
    its product with log2(e) are rounded once each, the constant is off by a
    quarter of a half step, so the exponent by 2.25 |t| half steps; the
    exponential by a step. Weighted with the probabilities |t| is at most
    ln V. Sums of positive terms are off by a half step for each addition
    that a term goes through, here at most 144."""
    return (2.25 * math.log(max(V, 2)) + 2 + 144) * HALF


def near(got, want, V):
    got, want = got.double().cpu().numpy(), want
    assert np.array_equal(np.isnan(got), np.isnan(want))
    same = np.isnan(want) | (got == want)
    off = np.abs(np.where(same, 0, got) - np.where(same, 0, want))
    assert np.all(off <= away(V) + HALF * np.where(same, 0, np.abs(want)))


def log_softmax64(x):
    x = x.double().cpu().numpy()
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        return (x - m) - np.log(np.exp(x - m).sum(1, keepdims=True))


def beams64(logits, scores, k):
    x = logits.double().cpu().numpy()
    c = scores.double().cpu().numpy()
    G, B = c.shape
    lp = log_softmax64(logits).reshape(G, B, -1)
    out = np.full((G, k), -INF), np.full((G, k), -1), np.full((G, k), -1)
    for g in range(G):
        total = c[g][:, None] + lp[g]
        b, t = np.nonzero(np.isfinite(total)
                          & np.isfinite(c[g])[:, None])
        first = np.lexsort((t, -x[g * B + b, t], b, -total[b, t]))[:k]
        n = len(first)
        out[0][g, :n] = total[b[first], t[first]]
        out[1][g, :n], out[2][g, :n] = b[first], t[first]
    return out


def rows_of(kind, R, V, dtype, device, pad=0, start=0, seed=0):
    """Rows of logits cut from wider ones, from a column on."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * 3
    if kind == "steps":        # many equal ones
        x = torch.randint(0, 3, (R, V), generator=g).float()
    elif kind == "equal":
        x = torch.full((R, V), 0.5)
    elif kind == "zeros":      # zeros of both signs are equal
        x = torch.where(x > 0, 0.0, -0.0)
    elif kind == "masked":
        x = x.masked_fill(torch.rand(R, V, generator=g) < 0.99, -INF)
    elif kind == "lowest":
        x = x.masked_fill(torch.rand(R, V, generator=g) < 0.99,
                          torch.finfo(dtype).min)
    elif kind == "gone":       # rows with no distribution among others
        x[::3] = -INF
        x[1::5, V // 2] = float("nan")
        x[2::7, V - 1] = INF
    elif kind == "large":
        x = x * 1e30
    elif kind == "clustered":  # large ones in few places of those at once
        t = torch.arange(V) * dtype.itemsize // 16 % 64
        x[:, t < 10] += 20
    elif kind == "plateau":    # some above many equal ones
        x = torch.where(torch.rand(R, V, generator=g) * V < 150, x.abs() + 9,
                        -3.0)
    elif kind == "tiny":       # below the normal numbers, still in order
        x = x * 1e-40
    elif kind == "rising":
        x = torch.arange(V).float().repeat(R, 1) / V * 8
    wide = torch.full((R, V + pad + start), 77.0).to(dtype)
    wide[:, start:start + V] = x.to(dtype)
    return wide.to(device)[:, start:start + V]


KINDS = ["random", "steps", "equal", "zeros", "masked", "lowest", "gone",
         "large", "rising", "clustered", "plateau", "tiny"]


def scores_of(G, B, kind="", seed=1):
    g = torch.Generator().manual_seed(seed)
    s = -5 * torch.rand(G, B, generator=g)
    if kind in ("steps", "equal", "zeros", "rising", "plateau", "tiny"):
        s[:] = -1.25
    if kind == "gone":
        s[0, 0] = -INF
    return s


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,B,V,k", [
    (1, 1, 1, 1), (1, 1, 1, 3), (2, 3, 2, 8), (7, 4, 9, 8), (3, 5, 1000, 10),
    (2, 32, 5003, 64), (33, 2, 2050, 4), (1, 4, 16385, 8), (2, 3, 33001, 1),
    (9, 8, 33001, 16), (9, 8, 33001, 230),
])
@pytest.mark.parametrize("kind", KINDS)
def test_beam_select(device, dtype, G, B, V, k, kind):
    if device == "cpu" and G * B * V > 100_000:
        pytest.skip("for the GPU")
    x = rows_of(kind, G * B, V, dtype, device, pad=3, start=1)
    c = scores_of(G, B, kind)
    got = ops.beam_select(x, c.to(device), k)
    s, p, t = beams64(x, c, k)
    assert got.scores.dtype == torch.float32
    assert got.parents.dtype == got.tokens.dtype == torch.int32
    assert np.array_equal(got.parents.cpu().numpy(), p)
    assert np.array_equal(got.tokens.cpu().numpy(), t)
    near(got.scores, s, V)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,k", [
    (1, 1, 0), (1, 1, 1), (3, 2, 2), (65, 9, 5), (4, 200, 200), (5, 1000, 20),
    (2, 5003, 129), (2, 5003, 256), (70, 16390, 256), (257, 2050, 1), (3, 16385, 0), (2, 33001, 5),
])
@pytest.mark.parametrize("kind", KINDS)
def test_top_logprobs(device, dtype, R, V, k, kind):
    x = rows_of(kind, R, V, dtype, device, pad=2, start=3)
    given = torch.arange(R, dtype=torch.int64 if V % 2 else torch.int32) \
        * 7919 % (V + 2) - 1          # -1 and V are among them
    got = ops.top_logprobs(x, k, given.to(device))
    lp, raw = log_softmax64(x), x.double().cpu().numpy()
    gone = np.isnan(lp).any(1)
    want = np.stack([np.arange(V) if gone[r] else
                     np.lexsort((np.arange(V), -raw[r])) for r in range(R)])
    want = want[:, :k]
    assert got.ids.dtype == torch.int32 and got.logprobs.shape == (R, k)
    assert np.array_equal(got.ids.cpu().numpy(), want)
    near(got.logprobs, np.take_along_axis(lp, want, 1), V)
    inside = (given >= 0) & (given < V)
    of = np.where(inside, lp[np.arange(R), given.clamp(0, V - 1)], -INF)
    near(got.token_logprobs, np.where(gone, np.nan, of), V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_vocabulary_and_many_rows(dtype):
    x = rows_of("random", 24, 151936, dtype, "cuda", seed=3)
    c = scores_of(3, 8)
    got = ops.beam_select(x, c.cuda(), 16)
    s, p, t = beams64(x, c, 16)
    assert np.array_equal(got.parents.cpu().numpy(), p)
    assert np.array_equal(got.tokens.cpu().numpy(), t)
    near(got.scores, s, x.shape[1])
    # rows by themselves and among thousands are the same
    many = x[:2].repeat(700, 1)
    top = ops.top_logprobs(many, 5)
    alone = ops.top_logprobs(x[:2], 5)
    assert torch.equal(top.ids, alone.ids.repeat(700, 1))
    near(top.logprobs, alone.logprobs.double().cpu().numpy()
         .repeat(1, 0)[np.arange(1400) % 2], x.shape[1])


@pytest.mark.parametrize("device", DEVICES)
def test_most_choices_of_one_row(device):
    x = rows_of("random", 2, 3001, torch.float32, device)
    got = ops.beam_select(x, torch.zeros(1, 2, device=device),
                          ops.MOST_CHOICES)
    s, p, t = beams64(x, torch.zeros(1, 2), ops.MOST_CHOICES)
    assert np.array_equal(got.tokens.cpu().numpy(), t)
    assert np.array_equal(got.parents.cpu().numpy(), p)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,integer,nan", [
    (torch.float32, torch.int32, 0x7f810000),
    (torch.bfloat16, torch.int16, 0x7f81)])
@pytest.mark.parametrize("k", [1, 20, 100, 230])
def test_signaling_nans_before_many_large_logits(device, dtype, integer, nan, k):
    """They may hide the logits beside them from a maximum, so that more than
    k are larger than what is found to be the largest."""
    x = rows_of("random", 6, 20000, dtype, "cpu", pad=3, start=1)
    want = ops.top_logprobs(x.to(device), k)
    c = scores_of(2, 3)
    c[1, 2] = -INF
    beams = ops.beam_select(x.to(device), c.to(device), k)
    pieces = x[5, :20000].unfold(0, 16 // dtype.itemsize, 16 // dtype.itemsize)
    pieces[::3] += 50
    pieces[::3, -1] = torch.tensor([nan], dtype=integer).view(dtype)
    assert torch.isnan(x[5]).any()
    got = ops.top_logprobs(x.to(device), k)
    assert torch.equal(got.logprobs[:5], want.logprobs[:5])
    assert torch.equal(got.ids[:5], want.ids[:5])
    assert torch.isnan(got.logprobs[5]).all()
    assert got.ids[5].tolist() == list(range(k))
    c[1, 2] = -1.0
    for a, b in zip(ops.beam_select(x.to(device), c.to(device), k), beams):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("k", [8, 60])
def test_long_beams(device, k):
    """Scores far below what one token adds or takes."""
    x = rows_of("random", 16, 2500, torch.bfloat16, device)
    c = -30000 + scores_of(2, 8)
    got = ops.beam_select(x, c.to(device), k)
    s, p, t = beams64(x, c, k)
    assert np.array_equal(got.parents.cpu().numpy(), p)
    assert np.array_equal(got.tokens.cpu().numpy(), t)
    near(got.scores, s, 2500)


@pytest.mark.parametrize("device", DEVICES)
def test_scores_cut_from_the_last_choice(device):
    """As a search goes on: the first B of its 2B candidates."""
    x = rows_of("random", 12, 501, torch.bfloat16, device)
    first = ops.beam_select(x, torch.zeros(3, 4, device=device), 8)
    c = first.scores[:, :4]
    assert not c.is_contiguous()
    got = ops.beam_select(x, c, 8)
    s, p, t = beams64(x, c.cpu(), 8)
    assert np.array_equal(got.tokens.cpu().numpy(), t)
    assert np.array_equal(got.parents.cpu().numpy(), p)
    turned = x.t().contiguous().t()   # tokens of a row far apart
    again = ops.beam_select(turned, c, 8)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows(device):
    x = torch.empty(0, 50, device=device)
    got = ops.beam_select(x, torch.empty(0, 4, device=device), 8)
    assert got.scores.shape == got.parents.shape == (0, 8)
    top = ops.top_logprobs(x, 3, torch.empty(0, dtype=torch.int32,
                                             device=device))
    assert top.ids.shape == (0, 3) and top.token_logprobs.shape == (0,)
    assert ops.top_logprobs(x, 0).token_logprobs is None


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.zeros(4, 10, device=device)
    c = torch.zeros(2, 2, device=device)
    ids = torch.zeros(4, dtype=torch.int32, device=device)
    for call in [
        lambda: ops.beam_select(x, c, 0),
        lambda: ops.beam_select(x, c, ops.MOST_CHOICES + 1),
        lambda: ops.beam_select(x.half(), c, 2),
        lambda: ops.beam_select(x[0], c, 2),
        lambda: ops.beam_select(x[:, :0], c, 2),
        lambda: ops.beam_select(x[:3], c, 2),
        lambda: ops.beam_select(x, c.double(), 2),
        lambda: ops.beam_select(x, c.view(-1), 2),
        lambda: ops.beam_select(x[:0], c[:, :0], 2),
        lambda: ops.beam_select(
            x.new_zeros(ops.MOST_BEAMS + 1, 3),
            x.new_zeros(1, ops.MOST_BEAMS + 1), 2),
        lambda: ops.beam_select(
            x.new_zeros(256, 1).expand(256, 163_841), x.new_zeros(1, 256), 2),
        lambda: ops.top_logprobs(x, 11),
        lambda: ops.top_logprobs(x, -1),
        lambda: ops.top_logprobs(x.double(), 2),
        lambda: ops.top_logprobs(x, 2, ids[:3]),
        lambda: ops.top_logprobs(x, 2, ids.float()),
        lambda: ops.copy_blocks_([x.t()], ids, ids),
        lambda: ops.copy_blocks_([x], ids.long(), ids),
        lambda: ops.copy_blocks_([x], ids, ids[:2]),
        lambda: ops.copy_blocks_([x], ids.view(2, 2), ids.view(2, 2)),
        lambda: ops.copy_blocks_([x], ids, ids, ids),
        lambda: ops.copy_blocks_([x.view(2, 2, 2, 5)], ids, ids, ids[:1]),
        lambda: ops.copy_blocks_([x.view(2, 2, 2, 5), x.view(2, 2, 5, 2)],
                                 ids, ids, ids),
    ]:
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_refuses_operands_apart():
    x, c = torch.zeros(4, 10, device="cuda"), torch.zeros(2, 2)
    ids = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.beam_select(x, c, 2)
    with pytest.raises(ValueError):
        ops.top_logprobs(x, 2, ids)
    with pytest.raises(ValueError):
        ops.copy_blocks_([x], ids, ids)


# -------------------------------------------------------- copies of blocks

def copied(tensors, src, dst, tokens=None):
    """Bytes of the tensors afterwards."""
    out = []
    for t in tensors:
        t = t.cpu().clone()
        old = t.clone()
        for i, (a, b) in enumerate(zip(src, dst)):
            if 0 <= a < len(t) and 0 <= b < len(t):
                if tokens is None:
                    t[b] = old[a]
                else:
                    n = min(max(tokens[i], 0), t.shape[2])
                    t[b, :, :n] = old[a, :, :n]
        out.append(t)
    return out


def same_bytes(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8),
                       b.cpu().contiguous().view(torch.uint8))


def bits(shape, dtype, device, seed, start=0):
    """Any bits, at an offset of `start` elements into the memory."""
    g = torch.Generator().manual_seed(seed)
    size = torch.empty((), dtype=dtype).element_size()
    n = math.prod(shape) + start
    raw = torch.randint(0, 256, (n * size,), generator=g, dtype=torch.uint8)
    return raw.to(device).view(dtype)[start:].view(shape)


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


SRC = [3, 3, 0, -1, 12, 8, 10 ** 9, 5, 7]
DST = [1, 2, 4, 6, 6, 13, 11, -5, 9]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tensors", [
    [((13, 8, 16, 128), torch.bfloat16, 0)] * 4,
    [((13, 2, 32, 128), torch.float8_e4m3fn, 0)] * 3,
    [((13, 1, 16, 288), torch.bfloat16, 0), ((13, 5, 16, 96), torch.float32, 1)],
    [((13, 3, 16, 3), torch.bfloat16, 1), ((13, 3, 16, 6), torch.bfloat16, 0)],
    [((13, 4, 16, 64), torch.uint8, 4)] * 101,
    [((13, 2, 16, 700), torch.float32, 0)],
])
@pytest.mark.parametrize("partly", [False, True])
def test_copy_pages(device, tensors, partly):
    ts = [bits(s, d, device, i, at) for i, (s, d, at) in enumerate(tensors)]
    tokens = [7, 16, 1, 5, 3, 2, 1, 4, 99] if partly else None
    src, dst = SRC, DST
    if partly:
        src, dst = src + [0, 0], dst + [10, 11]
        tokens = tokens + [0, -4]
    want = copied(ts, src, dst, tokens)
    ops.copy_blocks_(ts, ints(src, device), ints(dst, device),
                     ints(tokens, device) if partly else None)
    assert all(same_bytes(a, b) for a, b in zip(ts, want))


@pytest.mark.parametrize("device", DEVICES)
def test_copy_states(device):
    """Slots of any shape, down to a number each, beside large ones."""
    shapes = [(13,), (13, 3), (13, 3, 4096), (13, 16, 64, 64), (13, 0),
              (13, 7, 5)]
    ts = [bits(s, torch.float32, device, i) for i, s in enumerate(shapes)]
    ts.append(bits((13, 5), torch.uint8, device, 9))
    want = copied(ts, SRC, DST)
    ops.copy_blocks_(ts, ints(SRC, device), ints(DST, device))
    assert all(same_bytes(a, b) for a, b in zip(ts, want))


@pytest.mark.parametrize("device", DEVICES)
def test_copy_nothing(device):
    t = bits((4, 6), torch.float32, device, 0)
    old = t.clone()
    ops.copy_blocks_([t], ints([], device), ints([], device))
    ops.copy_blocks_([], ints([1], device), ints([2], device))
    assert torch.equal(t.view(torch.int32), old.view(torch.int32))


@pytest.mark.gpu
def test_copy_beyond_32_bits_of_offset():
    t = torch.zeros(40, 1, 16, 1 << 22, dtype=torch.bfloat16, device="cuda")
    t[39, :, :, :7] = 3.0
    t[39, :, :, -7:] = 5.0
    ops.copy_blocks_([t], ints([39, 39], "cuda"), ints([1, 38], "cuda"))
    for i in (1, 38):
        assert torch.equal(t[i, :, :, :9], t[39, :, :, :9])
        assert torch.equal(t[i, :, :, -9:], t[39, :, :, -9:])
    assert not t[2:38].any() and not t[0].any()


# ------------------------------------------------------- streams and graphs

@pytest.mark.gpu
def test_on_another_stream():
    x = rows_of("random", 8, 40000, torch.bfloat16, "cuda")
    c = scores_of(2, 4).cuda()
    want = ops.beam_select(x, c, 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        late = torch.empty_like(x)
        for _ in range(20):
            late.copy_(x)
        got = ops.beam_select(late, c, 8)
        top = ops.top_logprobs(late, 3, got.tokens.view(-1)[:8])
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    plain = ops.top_logprobs(x, 3, want.tokens.view(-1)[:8])
    assert all(torch.equal(a, b) for a, b in zip(top, plain))


@pytest.mark.gpu
def test_replayed_graphs():
    """Two graphs of a step (choice, copies by it, log-probabilities), replayed
    in turn on new inputs with other work between."""
    x = rows_of("random", 8, 40000, torch.bfloat16, "cuda").clone()
    c = scores_of(2, 4).cuda()
    pages = bits((64, 2, 16, 64), torch.bfloat16, "cuda", 0)
    dst = ints(list(range(40, 56)), "cuda")

    def step():
        got = ops.beam_select(x, c, 8)
        ops.copy_blocks_([pages], got.parents.view(-1), dst,
                         got.tokens.view(-1) % 17)
        return got, ops.top_logprobs(x, 5, got.tokens[:, :4].reshape(-1))

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    start = pages.clone()
    for i in range(6):
        graph, out = graphs[i % 2]
        x.copy_(rows_of("random", 8, 40000, torch.bfloat16, "cuda", seed=i))
        c.copy_(scores_of(2, 4, seed=i))
        pages.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        after = pages.clone()
        got, top = [[t.clone() for t in o] for o in out]
        pages.copy_(start)
        want, wtop = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(top, wtop))
        assert same_bytes(after, pages)


@pytest.mark.gpu
def test_same_again():
    x = rows_of("random", 64, 50021, torch.float32, "cuda")
    c = scores_of(8, 8).cuda()
    first = ops.beam_select(x, c, 16)
    for _ in range(5):
        assert all(torch.equal(a, b)
                   for a, b in zip(first, ops.beam_select(x, c, 16)))


# ------------------------------------------------- joins of many lists

def alone_at(x, c, k, first):
    """beams64 of the one search whose beams before `first` have no
    continuation."""
    s, p, t = beams64(x[first:], c[:, first:], k)
    return s, np.where(p < 0, p, p + first), t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["random", "steps"])
@pytest.mark.parametrize("k", [1, 16, 100, 256])
def test_last_beams_alone_go_on(dtype, kind, k):
    """256 beams of ten chunks each: those whose first choices a join reads
    first, 204 or more, have ended or no distribution."""
    V = 9 * 32768 // dtype.itemsize + 1
    x = rows_of(kind, 256, V, dtype, "cuda")
    c = scores_of(1, 256)
    c[0, :100] = -INF
    x[100:180, 5] = float("nan")
    x[180:230] = -INF
    c[0, 230:253] = -INF
    got = ops.beam_select(x, c.cuda(), k)
    s, p, t = alone_at(x, c, k, 253)
    assert np.array_equal(got.parents.cpu().numpy(), p)
    assert np.array_equal(got.tokens.cpu().numpy(), t)
    near(got.scores, s, V)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2, 9, 20000])
def test_no_probability_above_one(device, dtype, V):
    """Rows that all but one token are masked in, whatever its logit is: the
    sum is that token's term, and nothing rounds its log-probability above 0
    or a score above its beam's."""
    R = 2000 if V < 1000 else 64
    g = torch.Generator().manual_seed(V)
    at = torch.arange(R) * 7919 % V
    x = torch.full((R, V), -INF)
    x[torch.arange(R), at] = torch.randn(R, generator=g) * 30
    x = x.to(dtype).to(device)
    top = ops.top_logprobs(x, 1, at.to(device))
    assert torch.equal(top.ids.view(-1).long().cpu(), at)
    for lp in (top.logprobs.view(-1), top.token_logprobs):
        assert (lp <= 0).all() and (lp >= -away(1)).all()
    c = scores_of(R // 2, 2).to(device)
    best = ops.beam_select(x, c, 2)
    of = torch.gather(c, 1, best.parents.long())
    assert (best.scores <= of).all()


@pytest.mark.gpu
def test_refused_copies_copy_nothing():
    """A block of 2 GiB behind more tensors than one launch takes."""
    ts = [bits((2, 4), torch.float32, "cuda", i) for i in range(120)]
    old = [t.clone() for t in ts]
    ts.append(torch.empty(1, 1 << 31, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        ops.copy_blocks_(ts, ints([0], "cuda"), ints([1], "cuda"))
    assert all(same_bytes(a, b) for a, b in zip(ts, old))
    ops.copy_blocks_(ts, ints([], "cuda"), ints([], "cuda"))


def close(got, want, V):
    """As near(), for logits below 2^15 on a GPU. A term exp(t): the exponent
    t log2(e) is rounded once, |t| half steps, and the constant off by 0.23 of
    one, with |t| at most ln V on average; the exponential by a step. Three
    additions in 32 bits, then all in 64. A chunk's sum is scaled twice, each
    time by an exponential (a step) of an exponent below 0.5 (half a one)."""
    off = (1.23 * math.log(max(V, 2)) + 2 + 3 + 2 * 2.5) * HALF
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    some = np.isfinite(want)
    assert np.all(np.abs(got[some] - want[some])
                  <= off + HALF * np.abs(want[some]))


def first64(x, k):
    """Of rows on the GPU, without NaN: logits, log-probabilities and tokens of
    the k first, equal ones by token."""
    at = x.float().sort(dim=1, descending=True, stable=True).indices[:, :k]
    lp = torch.cat([torch.log_softmax(r.double(), 1) for r in x.split(32)])
    return [torch.gather(t, 1, at).double().cpu().numpy()
            for t in (x.float(), lp)] + [at.cpu().numpy()]


def one_search64(x, c, k):
    """beams64 of one search, by its beams' first tokens."""
    logit, lp, token = first64(x, k)
    beam = np.arange(len(x))[:, None].repeat(k, 1)
    s = c.double().numpy().reshape(-1, 1) + lp
    first = np.lexsort([a.reshape(-1) for a in (token, -logit, beam, -s)])[:k]
    return [a.reshape(-1)[first] for a in (s, beam, token)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,k", [
    (1, 151936, 20), (1, 151936, 0), (1, 151936, 256), (3, 1_000_003, 5),
    (2, 2_500_000, 64)])
@pytest.mark.parametrize("kind", ["random", "rising", "equal", "clustered"])
def test_rows_of_many_chunks(dtype, R, V, k, kind):
    """Up to 306 chunks a row, more than a wave has lanes; "rising": the last
    ones hold most of the sum and all choices."""
    x = rows_of(kind, R, V, dtype, "cuda", pad=1)
    given = torch.arange(R) * 7919 + V - 1 - R * 7919
    got = ops.top_logprobs(x, k, given.cuda())
    _, lp, token = first64(x, max(k, 1))
    assert np.array_equal(got.ids.cpu().numpy(), token[:, :k])
    close(got.logprobs, lp[:, :k], V)
    lp = torch.log_softmax(x.double(), 1).cpu()
    close(got.token_logprobs, lp[torch.arange(R), given].numpy(), V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["random", "steps", "equal", "plateau"])
@pytest.mark.parametrize("B,V,k", [
    (64, 41_000, 64), (64, 41_000, 256),        # 384 or 192 lists
    (256, 151_936, 16), (256, 151_936, 256)])   # 4864 or 2560
def test_one_search_of_many_lists(dtype, kind, B, V, k):
    """More lists than a join has threads, and than it reads at once."""
    x = rows_of(kind, B, V, dtype, "cuda")
    c = scores_of(1, B, kind)
    got = ops.beam_select(x, c.cuda(), k)
    s, b, t = one_search64(x, c, k)
    assert np.array_equal(got.parents.cpu().numpy()[0], b)
    assert np.array_equal(got.tokens.cpu().numpy()[0], t)
    close(got.scores[0], s, V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["random", "steps", "equal", "plateau",
                                  "clustered", "masked"])
@pytest.mark.parametrize("k", [33, 50, 64])
def test_many_choices_by_one_wave(dtype, kind, k):
    """Few chunks a row and more choices than half a wave's lanes."""
    x = rows_of(kind, 40, 50_021, dtype, "cuda", pad=2, start=1)
    got = ops.top_logprobs(x, k)
    _, lp, token = first64(x, k)
    assert np.array_equal(got.ids.cpu().numpy(), token)
    close(got.logprobs, lp, x.shape[1])
