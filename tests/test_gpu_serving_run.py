"""The operators over caller-held caches together, as a server runs them: a prompt's rows
go into the cache of a shared prefix, then each step writes the rows of the drafted
tokens, attends over prefix and own caches, verifies the drafts on the logits that
follow and keeps the accepted rows. Beside it the same run in numpy, 64-bit, on the
same logits; its attention reads its own record of the rows, not the caches.

Tolerance of the attention as derived for rn_attend_shared alone (test_gpu_serving_attend)."""
import numpy as np
import pytest
import torch

import rustyneedle_amd as rn
from test_gpu_serving_attend import Held, check as check_attention
from test_gpu_serving_cache import quantise
from test_gpu_serving_verify import rule

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, VOCAB, CAPACITY = 4, 200, 48


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=DEV)


def rows_of(k, v):
    return rn.CacheRows(rn.F32, k.data_ptr(), v.data_ptr(), *k.stride()[:3])


class Record(Held):
    """What the caches should hold: written rows in the format's numbers, kept on the side."""

    def __init__(self, format, sequences, kv, capacity):
        self.format, self.shape = format, (sequences, kv, capacity, 64)
        i8 = format == rn.CACHE_I8
        self.codes = [torch.zeros(self.shape, dtype=torch.int8 if i8 else torch.float16, device=DEV) for _ in range(2)]
        self.scales = [torch.ones(self.shape[:3], device=DEV) if i8 else None for _ in range(2)]

    def put(self, b, at, k, v):
        for i, x in enumerate((k, v)):  # x [tokens][kv][64]
            x = x.transpose(0, 1)
            if self.format == rn.CACHE_I8:
                codes, scale = quantise(x.cpu().numpy())  # (torch's device division by 127 is a product)
                self.scales[i][b, :, at:at + x.shape[1]] = torch.from_numpy(scale).to(DEV)
                x = torch.from_numpy(codes).to(DEV)
            self.codes[i][b, :, at:at + x.shape[1]] = x.to(self.codes[i].dtype)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("prefix_format,own_format", [(rn.CACHE_I8, rn.CACHE_I8), (rn.CACHE_F16, rn.CACHE_F16),
                                                      (rn.CACHE_F16, rn.CACHE_I8)])
@pytest.mark.parametrize("n,heads,kv,prefix", [(3, 4, 2, 37), (9, 8, 8, 1200)])
def test_a_server_of_drafted_tokens(n, heads, kv, prefix, prefix_format, own_format, graph):
    rng = np.random.default_rng(n)
    normal = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DEV)  # noqa: E731
    project = normal(heads * 64, VOCAB) * 0.2
    shared, own = rn.Cache(prefix_format, 1, kv, prefix), rn.Cache(own_format, n, kv, CAPACITY)
    shared_record, own_record = Record(prefix_format, 1, kv, prefix), Record(own_format, n, kv, CAPACITY)
    k, v = normal(1, prefix, kv, 64), normal(1, prefix, kv, 64)
    torch.cuda.synchronize()
    shared.write(rows_of(k, v), prefix)
    shared_record.put(0, 0, k[0], v[0])

    T = D + 1
    q, out = normal(n, T, heads, 64), torch.zeros((n, T, heads, 64), device=DEV)
    k, v = normal(n, T, kv, 64), normal(n, T, kv, 64)
    target, draft = torch.zeros((n, T, VOCAB), device=DEV), torch.zeros((n, D, VOCAB), device=DEV)
    starts, lengths, counts, drafted = ints([0] * n), ints([T] * n), ints([T] * n), ints([D] * n)
    tokens, uniforms = torch.zeros((n, D), dtype=torch.int32, device=DEV), torch.zeros((n, T), device=DEV)
    accepted, emitted, error = ints([0] * n), torch.full((n, T), -7, dtype=torch.int32, device=DEV), ints([0])
    size = rn.attend_shared_workspace(n, T, heads, shared, prefix, own)
    work = torch.empty((max(size, 1),), dtype=torch.uint8, device=DEV)
    judge = rn.verify_drafts_workspace(n, D, VOCAB)
    bench = torch.empty((max(judge, 1),), dtype=torch.uint8, device=DEV)

    def reads(stream):
        own.write(rows_of(k, v), T, starts.data_ptr(), counts.data_ptr(), error.data_ptr(), stream)
        rn.attend_shared(q.data_ptr(), out.data_ptr(), n, T, heads, shared, prefix, own, lengths.data_ptr(),
                         counts.data_ptr(), 0.125, 0, work.data_ptr(), size, error=error.data_ptr(), stream=stream)

    def judges(stream):
        rn.verify_drafts(n, D, VOCAB, target.data_ptr(), draft.data_ptr(), tokens.data_ptr(), drafted.data_ptr(), None,
                         uniforms.data_ptr(), accepted.data_ptr(), emitted.data_ptr(), None, bench.data_ptr(), judge,
                         error=error.data_ptr(), stream=stream)

    stream = torch.cuda.Stream()
    steps = [reads, judges]
    if graph:
        torch.cuda.synchronize()
        graphs = []
        for step in steps:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                step(stream.cuda_stream)
    held = np.zeros(n, int)  # rows each sequence keeps
    total = 0
    for turn in range(7):
        here = np.minimum(rng.integers(0, D + 1, n), CAPACITY - held - 1)  # drafts, and one token before them
        if (here < 0).any():
            break
        for t in (q, k, v):
            t.copy_(normal(*t.shape))
        starts.copy_(ints(held))
        counts.copy_(ints(here + 1))
        drafted.copy_(ints(here))
        lengths.copy_(ints(held + here + 1))
        uniforms.copy_(torch.from_numpy(rng.random((n, T), dtype=np.float32)))
        out.fill_(7.0)
        emitted.fill_(-7)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay() if graph else reads(stream.cuda_stream)
        torch.cuda.synchronize()
        for b in range(n):
            own_record.put(b, held[b], k[b, :here[b] + 1], v[b, :here[b] + 1])
        check_attention(out, q, shared_record, prefix, own_record, lengths, counts)

        target.copy_(out.reshape(n * T, heads * 64).mul(3).matmul(project).reshape(n, T, VOCAB))
        draft.copy_(target[:, :D] + 0.5 * normal(n, D, VOCAB))
        tokens.copy_(draft.argmax(-1).int())
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[1].replay() if graph else judges(stream.cuda_stream)
        torch.cuda.synchronize()
        kept, said = accepted.cpu().numpy(), emitted.cpu().numpy()
        for b in range(n):
            a, e, _ = rule(target[b].cpu().numpy(), draft[b].cpu().numpy(), tokens[b].cpu().numpy(), int(here[b]), 1.0,
                           uniforms[b].cpu().numpy(), VOCAB)
            assert kept[b] == a and said[b, :a + 1].tolist() == e, (turn, b)
        held += kept + 1
        total += int(kept.sum())
    assert turn > 3 and error.item() == 0 and total > 0

    # what the caches hold now, read back: code x scale, as recorded
    k, v = (torch.full((n, CAPACITY, kv, 64), 9.0, device=DEV) for _ in range(2))
    length = ints(held)
    torch.cuda.synchronize()
    own.read(rows_of(k, v), CAPACITY, None, length.data_ptr())
    torch.cuda.synchronize()
    for i, got in enumerate((k, v)):
        for b in range(n):
            want = own_record.codes[i][b, :, :held[b]].float()
            if own_format == rn.CACHE_I8:
                want = want * own_record.scales[i][b, :, :held[b], None]
            assert torch.equal(got[b, :held[b]], want.transpose(0, 1)), b
            assert (got[b, held[b]:] == 9.0).all()
