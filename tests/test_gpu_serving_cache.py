"""Rows written into caller-held caches and read back: codes and scales bit for bit
those of ops::quantise_int8 (rn_quantise_int8 and a numpy restatement of
ops.rs:103-118), fp16 rows rounded to nearest even, everything else left as it was."""
import numpy as np
import pytest
import torch

import rustyneedle_amd as rn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Held:
    """A cache's tensors with a sentinel in every element, in [sequences][kv][capacity] order or a stranger one."""

    def __init__(self, format, sequences, kv, capacity, order="contiguous"):
        gap = 3 if order != "contiguous" else 0
        if order == "heads first":
            self.head_rows, self.sequence_rows = sequences * (capacity + gap), capacity + gap
        else:
            self.head_rows = capacity + gap
            self.sequence_rows = kv * (capacity + gap) + 2 * gap
        rows = max(self.sequence_rows * sequences, self.head_rows * kv)
        kind = torch.int8 if format == rn.CACHE_I8 else torch.float16
        self.keys, self.values = (torch.full((rows, 64), 77, dtype=kind, device=DEV) for _ in range(2))
        self.key_scales, self.value_scales = (torch.full((rows,), 5.5, device=DEV) for _ in range(2))
        i8 = format == rn.CACHE_I8
        self.cache = rn.Cache.view(format, sequences, kv, capacity, self.keys.data_ptr(), self.values.data_ptr(),
                                   self.key_scales.data_ptr() if i8 else None,
                                   self.value_scales.data_ptr() if i8 else None, self.sequence_rows, self.head_rows)

    def at(self, b, h, position):
        return b * self.sequence_rows + h * self.head_rows + position


def device_rows(keys, values):
    """rn.CacheRows over tensors [sequences][tokens][kv][64] of any strides."""
    assert keys.stride() == values.stride()
    return rn.CacheRows(rn.F16 if keys.dtype == torch.float16 else rn.F32, keys.data_ptr(), values.data_ptr(),
                        *keys.stride()[:3])


def quantise(x):
    """ops.rs:103-118 in numpy, a row at a time."""
    x = x.astype(np.float32)
    with np.errstate(all="ignore"):
        peak = np.nanmax(np.where(np.isnan(x), 0, np.abs(x)), -1).astype(np.float32)
        scale = np.where(peak > 0, peak / np.float32(127), np.float32(1)).astype(np.float32)
        q = (x / scale[..., None]).astype(np.float32)
        code = np.clip(np.where(np.isnan(q), 0, np.rint(q)), -128, 127).astype(np.int8)
    return code, scale


def source(n, tokens, kv, kind, layout, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if layout == "fused":  # the q, k and v columns of one product
        x = torch.randn((n, tokens, 3, kv, 64), generator=g, device=DEV).to(kind)
        return x[:, :, 1], x[:, :, 2]
    k, v = (torch.randn((n, kv, tokens, 64), generator=g, device=DEV).to(kind) for _ in range(2))
    return k.transpose(1, 2), v.transpose(1, 2)


@pytest.mark.parametrize("order", ["contiguous", "gaps", "heads first"])
@pytest.mark.parametrize("kind,layout", [(torch.float32, "fused"), (torch.float16, "cache")])
@pytest.mark.parametrize("n,tokens,kv,capacity", [(1, 1, 1, 1), (3, 1, 4, 9), (2, 7, 3, 20), (5, 8, 2, 8), (2, 65, 1, 130),
                                                  (1, 600, 4, 1024)])
def test_write_and_read(n, tokens, kv, capacity, kind, layout, order):
    rng = np.random.default_rng(n + tokens)
    starts = rng.integers(0, capacity - tokens + 1, n)
    counts = rng.integers(0, tokens + 1, n)
    counts[0] = tokens
    starts_dev, counts_dev = ints(starts), ints(counts)
    k, v = source(n, tokens, kv, kind, layout)
    for format in (rn.CACHE_I8, rn.CACHE_F16):
        held = Held(format, n, kv, capacity, order)
        was = [t.clone() for t in (held.keys, held.values, held.key_scales, held.value_scales)]
        held.cache.write(device_rows(k, v), tokens, starts_dev.data_ptr(), counts_dev.data_ptr())
        torch.cuda.synchronize()
        want = [t.cpu().numpy() for t in was]
        for which, x in enumerate((k, v)):
            x = x.float().cpu().numpy()
            codes, scales = quantise(x)
            for b in range(n):
                for t in range(counts[b]):
                    for h in range(kv):
                        r = held.at(b, h, starts[b] + t)
                        if format == rn.CACHE_I8:
                            want[which][r], want[2 + which][r] = codes[b, t, h], scales[b, t, h]
                        else:
                            want[which][r] = x[b, t, h].astype(np.float16)
        got = [t.cpu().numpy() for t in (held.keys, held.values, held.key_scales, held.value_scales)]
        for a, b in zip(got, want):
            assert a.tobytes() == b.tobytes()
        # and back, into rows of both types that hold a sentinel past the counts
        for to in (torch.float32, torch.float16):
            out = [torch.full((n, kv, tokens, 64), 9.0, dtype=to, device=DEV).transpose(1, 2) for _ in range(2)]
            held.cache.read(device_rows(*out), tokens, starts_dev.data_ptr(), counts_dev.data_ptr())
            torch.cuda.synchronize()
            for which, o in enumerate(out):
                o = o.cpu().numpy()
                for b in range(n):
                    assert (o[b, counts[b]:] == 9.0).all()
                    for t in range(counts[b]):
                        for h in range(kv):
                            r = held.at(b, h, starts[b] + t)
                            row = want[which][r].astype(np.float32)
                            if format == rn.CACHE_I8:
                                row = row * want[2 + which][r]
                            assert np.array_equal(o[b, t, h], row.astype(o.dtype)), (b, t, h)


def test_write_equals_the_quantise_entry_point_on_strange_rows():
    """Zeros, subnormals, the largest floats, infinities and NaN, ties of the rounding."""
    x = np.zeros((12, 64), np.float32)
    x[1, 3] = -0.0
    x[2] = 1e-42
    x[3] = np.linspace(-3.4e38, 3.4e38, 64)
    x[4, 5] = np.inf
    x[5, 5], x[5, 6] = -np.inf, 2.0
    x[6, 7], x[6, 8] = np.nan, 3.0
    x[7] = np.nan
    x[8] = (np.arange(64) - 32) + 0.5
    x[8, 0] = 127.0
    x[9] = -np.arange(64) * np.float32(1e-38)
    x[10] = np.random.default_rng(0).standard_normal(64) * 1e-30
    x[11] = np.random.default_rng(1).standard_normal(64)
    codes, scales = rn.quantise_int8(x)
    d = torch.from_numpy(x).to(DEV).reshape(1, 12, 1, 64)
    held = Held(rn.CACHE_I8, 1, 1, 12)
    held.cache.write(device_rows(d, d), 12)
    torch.cuda.synchronize()
    for c, s in ((held.keys, held.key_scales), (held.values, held.value_scales)):
        assert np.array_equal(c.cpu().numpy(), codes)
        assert s.cpu().numpy().tobytes() == np.asarray(scales, np.float32).tobytes()


def test_numbers_out_of_range_leave_their_sequence_alone():
    n, tokens, capacity = 6, 4, 10
    k, v = source(n, tokens, 2, torch.float32, "fused")
    starts, counts, zeros = ints([0, -1, 7, 6, 0, 10]), ints([4, 4, 4, 4, 5, 0]), ints([0] * n)
    held, error = Held(rn.CACHE_I8, n, 2, capacity), ints([0])
    held.cache.write(device_rows(k, v), tokens, starts.data_ptr(), counts.data_ptr(), error.data_ptr())
    torch.cuda.synchronize()
    assert error.item() == rn.RN_ERR_ARGUMENT
    scales = held.key_scales.reshape(n, 2, capacity).cpu().numpy()
    written = (scales != 5.5).any(1)
    assert written.tolist() == [[True] * 4 + [False] * 6, [False] * 10, [False] * 10, [False] * 6 + [True] * 4,
                                [False] * 10, [False] * 10]
    # right numbers leave the word alone
    error.zero_()
    held.cache.write(device_rows(k, v), tokens, zeros.data_ptr(), None, error.data_ptr())
    out = [torch.full((n, tokens, 2, 64), 9.0, device=DEV) for _ in range(2)]
    held.cache.read(device_rows(*out), tokens, None, None, error.data_ptr())
    assert error.item() == 0
    held.cache.read(device_rows(*out), tokens, starts.data_ptr(), None, error.data_ptr())
    assert error.item() == rn.RN_ERR_ARGUMENT


def test_a_row_may_be_written_to_every_head():
    """Source strides of 0: one token's row for every sequence and head."""
    row = torch.randn((64,), device=DEV)
    rows = rn.CacheRows(rn.F32, row.data_ptr(), row.data_ptr(), 0, 0, 0)
    held = Held(rn.CACHE_F16, 3, 2, 5)
    held.cache.write(rows, 5)
    torch.cuda.synchronize()
    assert torch.equal(held.keys, row.half().expand(30, 64))


def test_positions_past_32_bits():
    """Rows whose element numbers need 64 bits: a batch's stride of 2^26 rows."""
    far = 1 << 26
    held = torch.zeros(((far + 2) * 64,), dtype=torch.int8, device=DEV)
    scales = torch.zeros((far + 2,), device=DEV)
    cache = rn.Cache.view(rn.CACHE_I8, 2, 1, 2, held.data_ptr(), held.data_ptr(), scales.data_ptr(), scales.data_ptr(),
                          far, 2)
    x = torch.randn((2, 2, 1, 64), device=DEV)
    cache.write(device_rows(x, x), 2)
    out = torch.zeros((2, 2, 1, 64), device=DEV)
    other = torch.zeros_like(out)
    cache.read(device_rows(out, other), 2)
    torch.cuda.synchronize()
    codes, s = quantise(x.cpu().numpy())
    assert np.array_equal(held[far * 64:].cpu().numpy().reshape(2, 64), codes[1, :, 0])
    assert np.array_equal(out.cpu().numpy(), codes * s[..., None])
    assert not held[128:far * 64].any()


def test_pointers_that_are_no_device_memory_are_refused():
    held, x = Held(rn.CACHE_I8, 1, 1, 4), torch.zeros((1, 4, 1, 64), device=DEV)
    host = np.zeros((1, 4, 1, 64), np.float32)
    for rows in (rn.CacheRows(rn.F32, host.ctypes.data & ~15, x.data_ptr(), 256, 64, 64),
                 rn.CacheRows(rn.F32, x.data_ptr() + 4, x.data_ptr(), 256, 64, 64)):
        with pytest.raises(rn.RnError) as e:
            held.cache.write(rows, 2)
        assert e.value.code == rn.RN_ERR_ARGUMENT
    with pytest.raises(rn.RnError):
        held.cache.write(device_rows(x, x), 2, host.ctypes.data & ~15)
    bad = rn.Cache.view(rn.CACHE_I8, 1, 1, 4, held.keys.data_ptr() + 8, held.values.data_ptr(),
                        held.key_scales.data_ptr(), held.value_scales.data_ptr())
    with pytest.raises(rn.RnError):
        bad.write(device_rows(x, x), 2)


def test_a_captured_write_follows_its_numbers():
    """A graph of a write and a read, replayed with other rows and positions, with eager work in between."""
    n, kv, capacity, tokens = 3, 2, 40, 5
    k, v = (torch.zeros((n, tokens, kv, 64), device=DEV) for _ in range(2))
    out = [torch.zeros_like(k) for _ in range(2)]
    starts = ints([0] * n)
    held = Held(rn.CACHE_I8, n, kv, capacity)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        held.cache.write(device_rows(k, v), tokens, starts.data_ptr(), None, None, stream.cuda_stream)
        held.cache.read(device_rows(*out), tokens, starts.data_ptr(), None, None, stream.cuda_stream)
    for step in range(4):
        a, b = source(n, tokens, kv, torch.float32, "fused", seed=step)
        k.copy_(a), v.copy_(b), starts.copy_(ints([step * tokens] * n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, o in zip((a, b), out):
            codes, s = quantise(x.cpu().numpy())
            assert np.array_equal(o.cpu().numpy(), codes * s[..., None]), step
    assert (held.key_scales.reshape(n, kv, capacity)[:, :, 20:] == 5.5).all()
