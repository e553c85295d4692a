"""rn_verify_drafts against the rule in 64 bits, a sequence and a token at a time:
whole numbers equal, probabilities within a rounding to f32 (2^-24) and 1e-9 of the
value (the 64-bit sums of both sides)."""
import numpy as np
import pytest
import torch

import rustyneedle_amd as rn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def device(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def address(t):
    return None if t is None else t.data_ptr()


def run(target, draft, tokens, counts, temperatures, uniforms, error=None, pad=0, stream=None):
    n, rows, vocab = target.shape
    d = rows - 1

    def padded(x):
        if x is None or not pad:
            return x
        wide = np.full(x.shape[:-1] + (vocab + pad,), np.nan, np.float32)
        wide[..., :vocab] = x
        return wide

    t, q = device(padded(target)), device(padded(draft))
    tok, cnt, temp, uni = device(tokens), device(counts), device(temperatures), device(uniforms)
    accepted = torch.full((n,), -7, dtype=torch.int32, device=DEV)
    emitted = torch.full((n, rows), -7, dtype=torch.int32, device=DEV)
    chance = torch.full((n, rows), -7.0, device=DEV)
    size = rn.verify_drafts_workspace(n, d, vocab)
    work = torch.full((size,), 0xff, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    rn.verify_drafts(n, d, vocab, t.data_ptr(), address(q), address(tok), address(cnt), address(temp), uni.data_ptr(),
                     accepted.data_ptr(), emitted.data_ptr(), chance.data_ptr(), work.data_ptr(), size, vocab + pad,
                     vocab + pad, address(error), stream)
    torch.cuda.synchronize()
    return accepted.cpu().numpy(), emitted.cpu().numpy(), chance.cpu().numpy()


def distribution(row, temperature):
    """softmax(row / temperature) in float64, or None where the row has none."""
    x = row.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return None
    if temperature == 0:
        p = np.zeros_like(x)
        p[np.argmax(x)] = 1.0
        return p
    p = np.exp((x - x.max()) / temperature)
    return p / p.sum()


def rule(target, draft, tokens, count, temperature, uniforms, vocab):
    """(accepted, emitted tokens, their probabilities) of one sequence."""
    out, chances = [], []
    d = target.shape[0] - 1
    if not 0 <= count <= d or not (0 <= temperature < np.inf):
        return 0, [-1], [0.0]
    for i in range(count + 1):
        p = distribution(target[i], temperature)
        if p is None:
            return i, out + [-1], chances + [0.0]
        if i == count:
            rest = p
            break
        x = tokens[i]
        q = np.zeros(vocab)
        if not 0 <= x < vocab:
            return i, out + [-1], chances + [0.0]
        if draft is None:
            q[x] = 1.0
        else:
            q = distribution(draft[i], temperature)
            if q is None:
                return i, out + [-1], chances + [0.0]
        taken = p[x] == 1.0 if temperature == 0 else float(uniforms[i]) * q[x] < p[x]
        if not taken:
            rest = np.maximum(p - q, 0.0)
            if temperature == 0 or not rest.sum() > 0:
                rest = p
            break
        out.append(int(x))
        chances.append(p[x])
    sums = np.cumsum(rest)
    over = np.nonzero((sums > float(uniforms[d]) * sums[-1]) & (rest > 0))[0]
    choice = int(over[0]) if len(over) else int(np.nonzero(rest > 0)[0][-1])
    return len(out), out + [choice], chances + [p[choice]]


def check(target, draft, tokens, counts, temperatures, uniforms, pad=0):
    n, rows, vocab = target.shape
    accepted, emitted, chance = run(target, draft, tokens, counts, temperatures, uniforms, pad=pad)
    for b in range(n):
        a, e, c = rule(target[b], None if draft is None else draft[b], None if tokens is None else tokens[b],
                       rows - 1 if counts is None else int(counts[b]),
                       1.0 if temperatures is None else float(temperatures[b]), uniforms[b], vocab)
        assert accepted[b] == a, (b, accepted[b], a)
        assert emitted[b, :a + 1].tolist() == e, (b, emitted[b], e)
        assert (emitted[b, a + 1:] == -7).all() and (chance[b, a + 1:] == -7).all(), "entries behind the run"
        assert np.allclose(chance[b, :a + 1], c, rtol=2.0 ** -24 + 1e-9, atol=1e-45), (b, chance[b], c)
    return accepted


def made(n, d, vocab, seed, near=0.7, temperature=None):
    rng = np.random.default_rng(seed)
    target = (3 * rng.standard_normal((n, d + 1, vocab))).astype(np.float32)
    draft = (target[:, :d] + near * rng.standard_normal((n, d, vocab))).astype(np.float32)
    temperatures = rng.uniform(0.5, 1.5, n).astype(np.float32)
    tokens = np.zeros((n, d), np.int32)
    for b in range(n):
        for i in range(d):
            tokens[b, i] = rng.choice(vocab, p=distribution(draft[b, i], temperatures[b]))
    uniforms = rng.random((n, d + 1), dtype=np.float32)
    return target, draft, tokens, temperatures, uniforms, rng


@pytest.mark.parametrize("n,d,vocab", [(1, 0, 1), (1, 1, 1), (2, 1, 2), (3, 2, 3), (5, 4, 101), (1, 4, 8192), (7, 3, 1023),
                                       (4, 5, 1024), (4, 5, 1025), (70, 4, 5001), (2, 63, 300), (300, 2, 50),
                                       (64, 8, 20000), (3, 0, 70001)])
def test_runs(n, d, vocab):
    target, draft, tokens, temperatures, uniforms, rng = made(n, d, vocab, n + d)
    accepted = check(target, draft, tokens, None, temperatures, uniforms)
    if n * d > 100 and vocab > 2:
        assert 0 < accepted.mean() < d  # both ends of the rule are met
    counts = rng.integers(0, d + 1, n).astype(np.int32)
    check(target, draft, tokens, counts, temperatures, uniforms, pad=3)
    check(target, None, tokens, counts, None, uniforms, pad=1)
    target[rng.random(target.shape) < 0.5] = -np.inf
    target[..., vocab // 2] = 0.5
    check(target, draft, tokens, counts, temperatures, uniforms)


@pytest.mark.parametrize("n,d,vocab", [(1, 0, 1), (6, 4, 37), (50, 3, 4099)])
def test_greedy(n, d, vocab):
    """Temperature 0: the first index of the maximum, whatever the uniforms; among warm sequences."""
    target, draft, _, temperatures, uniforms, rng = made(n, d, vocab, 3 * n)
    target = np.round(target)  # ties
    tokens = np.where(rng.random((n, d)) < 0.8, target[:, :d].argmax(-1), rng.integers(0, vocab, (n, d))).astype(np.int32)
    temperatures[rng.random(n) < 0.7] = 0.0
    temperatures[0] = 0.0
    for q in (draft, None):
        check(target, q, tokens, None, temperatures, uniforms)
    accepted, emitted, chance = run(target, None, tokens, None, np.zeros(n, np.float32), uniforms)
    for b in range(n):
        best = target[b].argmax(-1)
        a = next((i for i in range(d) if tokens[b, i] != best[i]), d)
        assert accepted[b] == a and emitted[b, :a + 1].tolist() == best[:a + 1].tolist()
        assert (chance[b, :a + 1] == 1.0).all()


def test_uniforms_at_their_ends():
    """0 accepts whatever the target may say; next to 1 the draw takes the last index with a weight."""
    target, draft, tokens, temperatures, uniforms, _ = made(40, 3, 200, 9)
    most = np.nextafter(np.float32(1), np.float32(0))
    for accept in (0.0, most):
        for drawn in (0.0, most):
            u = np.full_like(uniforms, accept)
            u[:, -1] = drawn
            check(target, draft, tokens, None, temperatures, u)
    target[:, :, 150:] = -np.inf
    check(target, draft, np.minimum(tokens, 149), None, temperatures, u)


def test_the_same_model_drafting_accepts_everything():
    target, _, tokens, temperatures, uniforms, _ = made(30, 5, 900, 10)
    accepted = check(target, target[:, :5].copy(), tokens, None, temperatures, uniforms)
    assert (accepted == 5).all()
    # a drafted token that neither may say is refused, and nothing is left of p - q: all of p is drawn from
    target[:, 0, 7] = -np.inf
    tokens[:, 0] = 7
    accepted = check(target, target[:, :5].copy(), tokens, None, temperatures, uniforms)
    assert (accepted == 0).all()


@pytest.mark.parametrize("size", [1e-3, 300.0, 1e30])
def test_logits_of_any_size(size):
    target, draft, tokens, temperatures, uniforms, _ = made(20, 2, 333, 11)
    check((target * size).astype(np.float32), (draft * size).astype(np.float32), tokens, None, temperatures, uniforms)


@pytest.mark.parametrize("n,vocab", [(3, 50), (40, 3000), (20, 20000)])
def test_masks_of_the_lowest_number(n, vocab):
    """Tokens masked with the lowest float: nothing where others are left, alike where all are."""
    target, draft, tokens, temperatures, uniforms, rng = made(n, 3, vocab, 31)
    lowest = np.finfo(np.float32).min
    out = rng.random(target.shape) < 0.7
    out[..., vocab // 3] = False
    target[out] = lowest
    target[1] = lowest
    draft[2] = lowest
    check(target, draft, tokens, None, temperatures, uniforms)
    check(target, None, tokens, None, temperatures, uniforms)


def test_rows_past_32_bits():
    """Rows of logits that lie more than 2^32 bytes apart."""
    vocab, apart = 300, (1 << 30) + 1
    target, draft, tokens, temperatures, uniforms, _ = made(1, 1, vocab, 33)
    wide = torch.empty((apart + vocab,), device=DEV)
    for i in range(2):
        wide[i * apart:i * apart + vocab] = device(target[0, i])
    q, tok, temp, uni = device(draft), device(tokens), device(temperatures), device(uniforms)
    accepted = torch.full((1,), -7, dtype=torch.int32, device=DEV)
    emitted = torch.full((1, 2), -7, dtype=torch.int32, device=DEV)
    size = rn.verify_drafts_workspace(1, 1, vocab)
    work = torch.zeros((size,), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    rn.verify_drafts(1, 1, vocab, wide.data_ptr(), q.data_ptr(), tok.data_ptr(), None, temp.data_ptr(), uni.data_ptr(),
                     accepted.data_ptr(), emitted.data_ptr(), None, work.data_ptr(), size, apart)
    torch.cuda.synchronize()
    a, e, _ = rule(target[0], draft[0], tokens[0], 1, float(temperatures[0]), uniforms[0], vocab)
    assert accepted.item() == a and emitted[0, :a + 1].tolist() == e


def test_what_cannot_be_judged_ends_the_run():
    n, d, vocab = 12, 3, 500
    target, draft, tokens, temperatures, uniforms, _ = made(n, d, vocab, 12)
    draft = target[:, :d].copy()  # everything is accepted up to the fault
    counts = np.full(n, d, np.int32)
    target[1, 2, 3] = np.nan
    target[2, 0, 499] = np.inf
    target[3, 3] = -np.inf
    draft[4, 1, 0] = np.nan
    draft[5, 0] = -np.inf
    tokens[6, 1], tokens[7, 2] = vocab, -1
    counts[8], counts[9] = -1, d + 1
    temperatures[10], temperatures[11] = -0.5, np.nan
    error = torch.zeros((1,), dtype=torch.int32, device=DEV)
    accepted, emitted, chance = run(target, draft, tokens, counts, temperatures, uniforms, error)
    assert error.item() == rn.RN_ERR_ARGUMENT
    ends = [d, 2, 0, 3, 1, 0, 1, 2, 0, 0, 0, 0]
    assert accepted.tolist() == ends
    for b in range(1, n):
        assert emitted[b, ends[b]] == -1 and chance[b, ends[b]] == 0.0
        assert emitted[b, :ends[b]].tolist() == tokens[b, :ends[b]].tolist()
    check(target, draft, tokens, counts, temperatures, uniforms)
    # faults behind the end of a run do not matter, nor do rows behind the count
    error.zero_()
    counts[:] = 0
    target, draft, tokens, temperatures, uniforms, _ = made(n, d, vocab, 13)
    target[:, 1:] = np.nan
    draft[:] = np.nan
    tokens[:] = -5
    run(target, draft, tokens, counts, temperatures, uniforms, error)
    assert error.item() == 0


def test_emitted_tokens_follow_the_target():
    """Whatever the draft proposes, the first emitted token has the target's
    distribution: 60000 sequences of the same logits, each frequency within six
    standard deviations."""
    n, vocab = 60000, 6
    rng = np.random.default_rng(14)
    one, other = rng.standard_normal((2, vocab)).astype(np.float32) * 1.5
    target = np.broadcast_to(one, (n, 2, vocab)).copy()
    draft = np.broadcast_to(other, (n, 1, vocab)).copy()
    p, q = distribution(one, 1.0), distribution(other, 1.0)
    tokens = rng.choice(vocab, size=(n, 1), p=q).astype(np.int32)
    uniforms = rng.random((n, 2), dtype=np.float32)
    accepted, emitted, _ = run(target, draft, tokens, None, None, uniforms)
    seen = np.bincount(emitted[:, 0], minlength=vocab) / n
    assert (np.abs(seen - p) < 6 * np.sqrt(p * (1 - p) / n)).all()
    assert abs(accepted.mean() - np.minimum(p, q).sum()) < 6 * 0.5 / np.sqrt(n)


def test_a_captured_verification():
    """A graph replayed over other logits and uniforms, against eager calls."""
    n, d, vocab = 9, 4, 3001
    first = made(n, d, vocab, 20)
    held = [device(x) for x in first[:5]]
    accepted = torch.zeros((n,), dtype=torch.int32, device=DEV)
    emitted = torch.zeros((n, d + 1), dtype=torch.int32, device=DEV)
    chance = torch.zeros((n, d + 1), device=DEV)
    size = rn.verify_drafts_workspace(n, d, vocab)
    work = torch.zeros((size,), dtype=torch.uint8, device=DEV)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        rn.verify_drafts(n, d, vocab, held[0].data_ptr(), held[1].data_ptr(), held[2].data_ptr(), None,
                         held[3].data_ptr(), held[4].data_ptr(), accepted.data_ptr(), emitted.data_ptr(),
                         chance.data_ptr(), work.data_ptr(), size, stream=stream.cuda_stream)
    for step in range(4):
        now = made(n, d, vocab, 21 + step)
        for h, x in zip(held, now[:5]):
            h.copy_(torch.from_numpy(x))
        emitted.fill_(-7), chance.fill_(-7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = run(now[0], now[1], now[2], None, now[3], now[4])
        for got, w in zip((accepted, emitted, chance), want):
            assert np.array_equal(got.cpu().numpy(), w), step


def test_pointers_that_are_no_device_memory_are_refused():
    target, draft, tokens, temperatures, uniforms, _ = made(2, 2, 50, 30)
    held = dict(target=device(target), draft=device(draft), tokens=device(tokens), uniforms=device(uniforms),
                accepted=torch.zeros(2, dtype=torch.int32, device=DEV),
                emitted=torch.zeros((2, 3), dtype=torch.int32, device=DEV),
                workspace=torch.zeros(1 << 16, dtype=torch.uint8, device=DEV))
    at = {k: v.data_ptr() for k, v in held.items()}

    def call(**wrong):
        a = dict(at, **wrong)
        rn.verify_drafts(2, 2, 50, a["target"], a["draft"], a["tokens"], None, None, a["uniforms"], a["accepted"],
                         a["emitted"], None, a["workspace"], 1 << 16)

    call()
    host = np.zeros(1024, np.float32)
    for name in at:
        with pytest.raises(rn.RnError) as e:
            call(**{name: (host.ctypes.data + 255) & ~255})
        assert e.value.code == rn.RN_ERR_ARGUMENT
    with pytest.raises(rn.RnError):
        call(workspace=at["workspace"] + 16)
