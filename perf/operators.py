"""The serving operators over caller-held device memory: what a pass of each reads
and returns, over the sizes that a server of this framework's models meets.

  write   the keys and values of new tokens into a batch's cache, and the written
          rows read back
  read    rows of a cache as floats
  attend  attention of a batch over one shared prefix and each sequence's own cache
  verify  drafted tokens against the target's probabilities, from given uniforms

listed() names twelve cases, draw() gives further ones of the same ranges,
prepare() makes what the user's program holds before the call, run() is one pass
(in elementary torch operations, or with `own` through the library), work() the
bytes and operations the pass cannot do without, exact() the same outputs in 64
bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
WIDTH = 64  # the head width of every model here


def listed():
    return [
        # one decode step of a small batch: each sequence's new row quantised into its cache (the smallest call)
        dict(name="write_step_16", op="write", format="i8", source="f32", sequences=16, tokens=1, kv_heads=4,
             capacity=1024, ragged=False),
        # the prompts of eight requests, from the fused q/k/v rows of a prefill
        dict(name="write_prompts_8x600", op="write", format="i8", source="f32", sequences=8, tokens=600, kv_heads=8,
             capacity=1024, ragged=True),
        # fp16 caches moved to 8 bits: sixteen long sequences
        dict(name="write_convert_16x4096", op="write", format="i8", source="f16", sequences=16, tokens=4096,
             kv_heads=8, capacity=4096, ragged=False),
        # one system prompt's cache read back to half precision
        dict(name="read_600_f16", op="read", format="i8", dest="f16", sequences=1, tokens=600, kv_heads=4,
             capacity=1024, ragged=False),
        # a batch's caches read back to floats
        dict(name="read_32x4096_f32", op="read", format="i8", dest="f32", sequences=32, tokens=4096, kv_heads=8,
             capacity=4096, ragged=True),
        # one decode step of a few chats over a system prompt (12 query heads on 4 key heads)
        dict(name="attend_16_prefix_600", op="attend", format="i8", sequences=16, queries=1, heads=12, kv_heads=4,
             prefix=600, longest=256, window=0),
        # an ordinary batch over a long fp16 prefix
        dict(name="attend_64_prefix_2048_f16", op="attend", format="f16", sequences=64, queries=1, heads=8,
             kv_heads=8, prefix=2048, longest=512, window=0),
        # drafted tokens of a batch attended together: up to five rows a sequence
        dict(name="attend_32x5_prefix_4096", op="attend", format="i8", sequences=32, queries=5, heads=12, kv_heads=4,
             prefix=4096, longest=512, window=0),
        # the largest: many sequences over one long document
        dict(name="attend_256_prefix_32768", op="attend", format="i8", sequences=256, queries=1, heads=8, kv_heads=8,
             prefix=32768, longest=1024, window=0),
        # one chat's four drafted tokens
        dict(name="verify_1x4", op="verify", sequences=1, drafts=4, vocab=8192, drafted=True, masked=False,
             greedy=False),
        # a batch's drafted tokens under a grammar, a few of the requests greedy
        dict(name="verify_64x4_masked", op="verify", sequences=64, drafts=4, vocab=8192, drafted=True, masked=True,
             greedy=True),
        # a large vocabulary
        dict(name="verify_64x8_65536", op="verify", sequences=64, drafts=8, vocab=65536, drafted=True, masked=False,
             greedy=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend", "attend", "verify", "verify"))
    kv_heads = rng.choice((1, 2, 4, 8))
    if op in ("write", "read"):
        while True:
            sequences, tokens = _log(rng, 1, 128), _log(rng, 1, 4096)
            if sequences * tokens * kv_heads <= 16 * 4096 * 8:
                break
        c = dict(op=op, format=rng.choice(("i8", "i8", "f16")), sequences=sequences, tokens=tokens, kv_heads=kv_heads,
                 capacity=tokens + _log(rng, 1, 1024), ragged=rng.random() < 0.5)
        c["source" if op == "write" else "dest"] = rng.choice(("f32", "f16"))
        return c
    if op == "attend":
        while True:
            heads = kv_heads * rng.choice((1, 2, 3, 4))
            sequences, queries = _log(rng, 1, 256), rng.choice((1, 1, 1, 2, 3, 5, 9))
            prefix, longest = rng.choice((0, _log(rng, 1, 32768), _log(rng, 64, 32768))), _log(rng, 16, 2048)
            if sequences * queries * heads * (prefix + longest) <= 256 * 8 * 33000 \
                    and sequences * kv_heads * longest <= 256 * 8 * 1024:
                break
        return dict(op=op, format=rng.choice(("i8", "i8", "f16")), sequences=sequences, queries=queries, heads=heads,
                    kv_heads=kv_heads, prefix=prefix, longest=longest, window=rng.choice((0, 0, 0, 1024, 200)))
    while True:
        sequences, drafts, vocab = _log(rng, 1, 128), rng.randrange(0, 9), _log(rng, 100, 131072)
        if sequences * (2 * drafts + 1) * vocab <= 64 * 17 * 65536:
            break
    return dict(op=op, sequences=sequences, drafts=drafts, vocab=vocab, drafted=rng.random() < 0.7,
                masked=rng.random() < 0.4, greedy=rng.random() < 0.4)


# ---- inputs ------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def _counts(rng, low, high, n):
    """Whole numbers of [low, high] on the device, one of them the highest."""
    out = rng.integers(low, high + 1, n).astype(np.int32)
    out[rng.integers(0, n)] = high
    return torch.from_numpy(out).to(DEVICE)


def _cache(g, fmt, sequences, kv_heads, capacity):
    """A filled cache: keys, values [sequences][kv_heads][capacity][64], in 8 bits
    with a scale a row (peak / 127 of rows of normal values)."""
    shape = (sequences, kv_heads, capacity, WIDTH)
    if fmt == "f16":
        return dict(format=fmt, keys=_normal(g, shape, torch.float16), values=_normal(g, shape, torch.float16),
                    key_scales=None, value_scales=None)

    def codes():
        return torch.randint(-127, 128, shape, generator=g, device=DEVICE, dtype=torch.int8)

    def scales():
        return (2.0 + torch.rand(shape[:3], generator=g, device=DEVICE)) / 127.0

    return dict(format=fmt, keys=codes(), values=codes(), key_scales=scales(), value_scales=scales())


def prepare(case, seed):
    c, g, rng = dict(case), _generator(seed), np.random.default_rng(seed)
    if c["op"] in ("write", "read"):
        n, t, h = c["sequences"], c["tokens"], c["kv_heads"]
        c["cache"] = _cache(g, c["format"], n, h, c["capacity"])
        c["starts"] = torch.from_numpy(rng.integers(0, c["capacity"] - t + 1, n).astype(np.int32)).to(DEVICE)
        c["counts"] = _counts(rng, (t + 1) // 2, t, n) if c["ragged"] else None
        kind = torch.float16 if c.get("dest") == "f16" else torch.float32
        c["out"] = [torch.zeros((n, h, t, WIDTH), device=DEVICE, dtype=kind) for _ in range(2)]
        if c["op"] == "write" and c["source"] == "f32":  # the fused rows of a product: q, k and v of every token
            rows = _normal(g, (n, t, 3, h, WIDTH))
            c["new"] = [rows[:, :, 1], rows[:, :, 2]]
        elif c["op"] == "write":  # another cache's rows
            c["new"] = [_normal(g, (n, h, t, WIDTH), torch.float16).transpose(1, 2) for _ in range(2)]
        return c
    if c["op"] == "attend":
        n, t = c["sequences"], c["queries"]
        c["q"] = _normal(g, (n, t, c["heads"], WIDTH))
        c["shared"] = _cache(g, c["format"], 1, c["kv_heads"], c["prefix"]) if c["prefix"] else None
        c["own_cache"] = _cache(g, c["format"], n, c["kv_heads"], c["longest"] + t)
        c["counts"] = _counts(rng, 1, t, n) if t > 1 else None
        c["lengths"] = _counts(rng, c["longest"] // 16 + t, c["longest"] + t, n)
        c["out"] = torch.zeros((n, t, c["heads"], WIDTH), device=DEVICE)
        return c
    n, d, vocab = c["sequences"], c["drafts"], c["vocab"]
    target = 3.0 * _normal(g, (n, d + 1, vocab))
    near = target[:, :d] + 0.7 * _normal(g, (n, d, vocab))  # a smaller model's logits
    temperatures = 0.5 + 0.7 * torch.rand((n,), generator=g, device=DEVICE)
    if c["greedy"]:
        temperatures = torch.where(torch.rand((n,), generator=g, device=DEVICE) < 0.3,
                                   torch.zeros_like(temperatures), temperatures)
    if c["masked"]:  # tokens that a grammar leaves out
        out = torch.rand((n, d + 1, vocab), generator=g, device=DEVICE) < 0.6
        out[:, :, 0] = False
        target.masked_fill_(out, float("-inf"))
    noise = -torch.log(-torch.log(torch.rand((n, d, vocab), generator=g, device=DEVICE).clamp_(1e-10, 1 - 1e-7)))
    warm = temperatures[:, None, None]
    pick = torch.where(warm > 0, near + warm * noise, near) if c["drafted"] else near
    c["target"], c["draft"] = target, near if c["drafted"] else None
    c["tokens"] = pick.argmax(-1).to(torch.int32) if d else torch.zeros((n, 0), device=DEVICE, dtype=torch.int32)
    c["temperatures"] = temperatures
    c["counts"] = _counts(rng, min(1, d), d, n) if c["greedy"] else None
    c["uniforms"] = torch.rand((n, d + 1), generator=g, device=DEVICE)
    c["accepted"] = torch.zeros((n,), device=DEVICE, dtype=torch.int32)
    c["emitted"] = torch.full((n, d + 1), -1, device=DEVICE, dtype=torch.int32)
    c["probabilities"] = torch.zeros((n, d + 1), device=DEVICE)
    return c


# ---- one pass ----------------------------------------------------------------------

def run(s):
    if own:
        return _run_library(s)
    if s["op"] == "write":
        _write(s)
        return _written(s, *_read(s))
    if s["op"] == "read":
        return dict(zip(("keys", "values"), _read(s)))
    if s["op"] == "attend":
        return _attend(s)
    return _verify(s)


def _written(s, keys, values):
    if s["format"] == "f16":
        return dict(keys=keys, values=values)
    return dict(keys=keys, values=values, key_scales=s["cache"]["key_scales"],
                value_scales=s["cache"]["value_scales"])


def _library_cache(rn, cache):
    """The library's view of a cache's tensors."""
    n, h, capacity, _ = cache["keys"].shape
    if cache["format"] == "f16":
        return rn.Cache.view(rn.CACHE_F16, n, h, capacity, cache["keys"].data_ptr(), cache["values"].data_ptr())
    return rn.Cache.view(rn.CACHE_I8, n, h, capacity, cache["keys"].data_ptr(), cache["values"].data_ptr(),
                         cache["key_scales"].data_ptr(), cache["value_scales"].data_ptr())


def _library_rows(rn, keys, values):
    """The library's view of rows [sequences][tokens][kv_heads][64]."""
    strides = keys.stride()
    return rn.CacheRows(rn.F16 if keys.dtype == torch.float16 else rn.F32, keys.data_ptr(), values.data_ptr(),
                        strides[0], strides[1], strides[2])


def _address(t):
    return None if t is None else t.data_ptr()


def _run_library(s):
    import rustyneedle_amd as rn
    if s["op"] in ("write", "read"):
        cache, counts = _library_cache(rn, s["cache"]), _address(s["counts"])
        starts = s["starts"].data_ptr()
        if s["op"] == "write":
            cache.write(_library_rows(rn, *s["new"]), s["tokens"], starts, counts)
        cache.read(_library_rows(rn, s["out"][0].transpose(1, 2), s["out"][1].transpose(1, 2)), s["tokens"], starts,
                   counts)
        return _written(s, *s["out"]) if s["op"] == "write" else dict(keys=s["out"][0], values=s["out"][1])
    if s["op"] == "attend":
        n, t, heads = s["sequences"], s["queries"], s["heads"]
        shared = _library_cache(rn, s["shared"]) if s["shared"] else None
        cache = _library_cache(rn, s["own_cache"])
        if "workspace" not in s:
            size = rn.attend_shared_workspace(n, t, heads, shared, s["prefix"], cache)
            s["workspace"] = torch.empty(size, device=DEVICE, dtype=torch.uint8)
        rn.attend_shared(s["q"].data_ptr(), s["out"].data_ptr(), n, t, heads, shared, s["prefix"], cache,
                         s["lengths"].data_ptr(), _address(s["counts"]), 1.0 / 8.0, s["window"],
                         s["workspace"].data_ptr(), s["workspace"].numel())
        return s["out"]
    n, d, vocab = s["sequences"], s["drafts"], s["vocab"]
    if "workspace" not in s:
        s["workspace"] = torch.empty(rn.verify_drafts_workspace(n, d, vocab), device=DEVICE, dtype=torch.uint8)
    rn.verify_drafts(n, d, vocab, s["target"].data_ptr(), _address(s["draft"]), s["tokens"].data_ptr(),
                     _address(s["counts"]), s["temperatures"].data_ptr(), s["uniforms"].data_ptr(),
                     s["accepted"].data_ptr(), s["emitted"].data_ptr(), s["probabilities"].data_ptr(),
                     s["workspace"].data_ptr(), s["workspace"].numel())
    return dict(accepted=s["accepted"], tokens=s["emitted"], probabilities=s["probabilities"])


# ---- the plain forms -----------------------------------------------------------------

def _places(s):
    """Index tensors of the rows [sequences][kv_heads][tokens], and which of them count."""
    at = torch.arange(s["tokens"], device=DEVICE)
    places = (torch.arange(s["sequences"], device=DEVICE)[:, None, None],
              torch.arange(s["kv_heads"], device=DEVICE)[None, :, None], s["starts"].long()[:, None, None] + at)
    return places, None if s["counts"] is None else (at < s["counts"][:, None])[:, None, :]


def _write(s):
    cache, (places, counted) = s["cache"], _places(s)

    def put(into, rows):
        into[places] = rows if counted is None else torch.where(
            counted if rows.dim() == 3 else counted[..., None], rows, into[places])

    for name, new in zip(("key", "value"), s["new"]):
        rows = new.transpose(1, 2)
        if s["format"] == "f16":
            put(cache[name + "s"], rows.to(torch.float16))
            continue
        rows = rows.float()
        peak = rows.abs().amax(-1)
        # tensors on both sides: a division by a number would multiply by its rounded reciprocal
        scale = torch.where(peak > 0, peak / torch.full_like(peak, 127.0), torch.ones_like(peak))
        put(cache[name + "s"], torch.clamp(torch.round(rows / scale[..., None]), -128, 127).to(torch.int8))
        put(cache[name + "_scales"], scale)


def _read(s):
    cache, (places, counted) = s["cache"], _places(s)
    got = []
    for name, out in zip(("key", "value"), s["out"]):
        rows = cache[name + "s"][places].float()
        if s["format"] == "i8":
            rows = rows * cache[name + "_scales"][places][..., None]
        rows = rows.to(out.dtype)
        got.append(rows if counted is None else torch.where(counted[..., None], rows, out))
    return got


def _floats(cache):
    keys, values = cache["keys"].float(), cache["values"].float()
    if cache["format"] == "i8":
        keys, values = keys * cache["key_scales"][..., None], values * cache["value_scales"][..., None]
    return keys, values


def _limits(s):
    """First and last + 1 position each row [sequences][queries] sees, over prefix and own cache."""
    n, t, prefix = s["sequences"], s["queries"], s["prefix"]
    counts = torch.full((n,), t, device=DEVICE) if s["counts"] is None else s["counts"].long()
    at = torch.arange(t, device=DEVICE)
    end = prefix + (s["lengths"].long() - counts)[:, None] + at + 1
    first = (end - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(end)
    return first, end, at < counts[:, None]


def _attend(s):
    n, t, kv, prefix = s["sequences"], s["queries"], s["kv_heads"], s["prefix"]
    group = s["heads"] // kv
    first, end, counted = _limits(s)
    q = s["q"].reshape(n, t, kv, group, WIDTH) * (1.0 / 8.0)
    by_sequence = q.permute(0, 2, 1, 3, 4).reshape(n, kv, t * group, WIDTH)
    keys, values = _floats(s["own_cache"])
    scores = torch.matmul(by_sequence, keys.transpose(2, 3).contiguous()).reshape(n, kv, t, group, -1)
    if prefix:
        pk, pv = _floats(s["shared"])
        by_head = q.permute(2, 0, 1, 3, 4).reshape(kv, n * t * group, WIDTH)
        over = torch.matmul(by_head, pk[0].transpose(1, 2).contiguous())
        scores = torch.cat([over.reshape(kv, n, t, group, prefix).transpose(0, 1), scores], -1)
    at = torch.arange(scores.shape[-1], device=DEVICE)
    seen = (at >= first[..., None]) & (at < end[..., None])
    scores = scores.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., prefix:].reshape(n, kv, t * group, -1), values).reshape(n, kv, t, group, WIDTH)
    if prefix:
        over = torch.matmul(p[..., :prefix].transpose(0, 1).reshape(kv, n * t * group, prefix), pv[0])
        out = out + over.reshape(kv, n, t, group, WIDTH).transpose(0, 1)
    out = (out / total).permute(0, 2, 1, 3, 4).reshape(n, t, s["heads"], WIDTH)
    return torch.where(counted[..., None, None], out, s["out"])


def _distribution(logits, temperatures):
    """softmax(logits / temperature) in 64 bits (the draw's border lies between sums of thousands of
    terms); at temperature 0 all of it on the first largest logit."""
    x = logits.double()
    peak = x.amax(-1, keepdim=True)
    warm = temperatures.double()[:, None, None]
    w = torch.exp((x - peak) / torch.where(warm > 0, warm, torch.ones_like(warm)))
    w = w / w.sum(-1, keepdim=True)
    ids = torch.arange(x.shape[-1], device=DEVICE)
    return torch.where(warm > 0, w, (ids == x.argmax(-1, keepdim=True)).double())


def _verify(s):
    n, d, vocab = s["sequences"], s["drafts"], s["vocab"]
    counts = torch.full((n,), d, device=DEVICE) if s["counts"] is None else s["counts"].long()
    p = _distribution(s["target"], s["temperatures"])
    tokens, u = s["tokens"].long()[..., None], s["uniforms"].double()
    ids = torch.arange(vocab, device=DEVICE)
    q = (ids == tokens).double() if s["draft"] is None else _distribution(s["draft"], s["temperatures"])
    at = torch.arange(d, device=DEVICE)
    good = u[:, :d] * q.gather(-1, tokens)[..., 0] < p[:, :d].gather(-1, tokens)[..., 0]
    accepted = torch.cumprod((good & (at < counts[:, None])).long(), 1).sum(1)
    rows = torch.arange(n, device=DEVICE)
    here = p[rows, accepted]
    rest = here
    if d:
        refused = accepted < counts
        left = torch.clamp(here - q[rows, accepted.clamp(max=d - 1)], min=0.0)
        rest = torch.where((refused & (left.sum(-1) > 0))[:, None], left, here)
    below = torch.cumsum(rest, -1) <= u[:, d, None] * rest.sum(-1, keepdim=True)
    last = torch.where(rest > 0, ids, torch.zeros_like(ids)).amax(-1)
    chosen = torch.minimum(below.sum(-1), last)
    emitted = torch.cat([s["tokens"].long(), chosen[:, None]], 1)
    place = torch.arange(d + 1, device=DEVICE)
    emitted = torch.where(place == accepted[:, None], chosen[:, None], emitted)
    chance = p.gather(-1, emitted[..., None])[..., 0].float()
    live = place <= accepted[:, None]
    return dict(accepted=accepted.to(torch.int32),
                tokens=torch.where(live, emitted.to(torch.int32), s["emitted"]),
                probabilities=torch.where(live, chance, s["probabilities"]))


# ---- the work of a pass ----------------------------------------------------------------

def work(case):
    c = case
    if c["op"] in ("write", "read"):
        rows = 2 * c["sequences"] * c["kv_heads"] * c["tokens"]
        rows = rows * 3 // 4 if c["ragged"] else rows
        held = WIDTH + 4 if c["format"] == "i8" else 2 * WIDTH
        moved = rows * held + rows * WIDTH * (2 if c.get("dest") == "f16" else 4)  # read: a cache row in, floats out
        if c["op"] == "write":  # a source row in, a cache row out, before that
            moved += rows * held + rows * WIDTH * (2 if c["source"] == "f16" else 4)
        return dict(bytes=moved, flops=rows * WIDTH * (6 if c["op"] == "write" else 1))
    if c["op"] == "attend":
        n, t, prefix = c["sequences"], c["queries"], c["prefix"]
        rows = n * ((t + 1) / 2 if t > 1 else 1)
        mean = c["longest"] * 17 / 32 + t  # the mean of the ragged lengths
        seen = min(c["window"], prefix + mean) if c["window"] else prefix + mean
        held = 2 * (WIDTH + 4) if c["format"] == "i8" else 4 * WIDTH  # a key and a value row
        mean_seen = min(mean, seen)
        return dict(bytes=c["kv_heads"] * held * (min(prefix, seen) + n * mean_seen)
                    + 8 * WIDTH * rows * c["heads"], flops=4 * WIDTH * rows * c["heads"] * seen)
    n, d, vocab = c["sequences"], c["drafts"], c["vocab"]
    rows = n * (d + 1 + (d if c["drafted"] else 0))
    return dict(bytes=4 * rows * vocab + n * (d + 1) * 16, flops=4 * rows * vocab)


# ---- the same outputs in 64 bits -----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("write", "read"):
        return _exact_rows(s)
    return _exact_attend(s) if s["op"] == "attend" else _exact_verify(s)


def _exact_rows(s):
    """A cache row holds clamp(round(x / scale)) with the scale peak / 127 kept in 32
    bits and the quotient rounded to 32 bits, as the cache's definition has it."""
    n, t = s["sequences"], s["tokens"]
    starts = s["starts"].tolist()
    counts = [t] * n if s["counts"] is None else s["counts"].tolist()
    result = {}
    for i, name in enumerate(("key", "value")):
        held = s["cache"][name + "s"].double()
        if s["format"] == "i8":
            scales = s["cache"][name + "_scales"].double()
            if s["op"] == "write":
                result[name + "_scales"] = scales
        out = torch.zeros(s["out"][i].shape, device=DEVICE, dtype=torch.float64)
        for b in range(n):
            a, z = starts[b], starts[b] + counts[b]
            if s["op"] == "write":
                x = s["new"][i][b, :counts[b]].transpose(0, 1).double()
                if s["format"] == "f16":
                    held[b, :, a:z] = x.float().half().double()
                else:
                    peak = x.abs().max(-1).values
                    scales[b, :, a:z] = torch.where(peak > 0, peak / 127.0, torch.ones_like(peak))
                    kept = scales[b, :, a:z, None].float().double()
                    held[b, :, a:z] = (x / kept).float().double().round().clamp(-128, 127)
            out[b, :, :counts[b]] = held[b, :, a:z]
            if s["format"] == "i8":
                out[b, :, :counts[b]] *= scales[b, :, a:z, None].float().double()
        result[name + "s"] = out
    return result


def _exact_attend(s):
    n, t, kv, prefix = s["sequences"], s["queries"], s["kv_heads"], s["prefix"]
    group = s["heads"] // kv

    def doubles(cache, b, h, length):
        k, v = cache["keys"][b, h, :length].double(), cache["values"][b, h, :length].double()
        if cache["format"] == "i8":
            k = k * cache["key_scales"][b, h, :length].double()[:, None]
            v = v * cache["value_scales"][b, h, :length].double()[:, None]
        return k, v

    lengths = s["lengths"].tolist()
    counts = [t] * n if s["counts"] is None else s["counts"].tolist()
    out = s["out"].double()
    for h in range(kv):
        heads = slice(h * group, (h + 1) * group)
        if prefix:
            pk, pv = doubles(s["shared"], 0, h, prefix)
        for b in range(n):
            k, v = doubles(s["own_cache"], b, h, lengths[b])
            if prefix:
                k, v = torch.cat([pk, k]), torch.cat([pv, v])
            q = s["q"][b, :counts[b], heads].double()
            scores = torch.matmul(q.reshape(-1, WIDTH), k.T) / 8.0
            position = torch.arange(prefix + lengths[b] - counts[b], prefix + lengths[b], device=DEVICE)
            behind = position[:, None] - torch.arange(prefix + lengths[b], device=DEVICE)
            hidden = behind < 0
            if s["window"]:
                hidden = hidden | (behind >= s["window"])
            scores.masked_fill_(hidden.repeat_interleave(group, 0), float("-inf"))
            out[b, :counts[b], heads] = torch.matmul(torch.softmax(scores, -1), v).reshape(-1, group, WIDTH)
    return out


def _exact_verify(s):
    """Each sequence's loop over its drafted tokens, as the rule is stated."""
    n, d = s["sequences"], s["drafts"]
    counts = [d] * n if s["counts"] is None else s["counts"].tolist()
    tokens, warm = s["tokens"].tolist(), s["temperatures"].double().tolist()
    uniforms = s["uniforms"].double().tolist()
    accepted = s["accepted"].clone()
    emitted, chances = s["emitted"].clone(), s["probabilities"].double()

    def chance(row, temperature):
        x = row.double()
        if temperature > 0:
            return torch.softmax(x / temperature, -1)
        one = torch.zeros_like(x)
        one[x.argmax()] = 1.0
        return one

    for b in range(n):
        i, rest = 0, None
        while True:
            p = chance(s["target"][b, i], warm[b])
            if i == counts[b]:
                rest = p
                break
            x = tokens[b][i]
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1.0
            else:
                q = chance(s["draft"][b, i], warm[b])
            if not uniforms[b][i] * float(q[x]) < float(p[x]):
                rest = torch.relu(p - q)
                rest = rest if float(rest.sum()) > 0 else p
                break
            emitted[b, i], chances[b, i] = x, p[x]
            i += 1
        sums = torch.cumsum(rest, 0)
        over = torch.nonzero((sums > uniforms[b][d] * float(rest.sum())) & (rest > 0))
        choice = int(over[0]) if len(over) else int(torch.nonzero(rest > 0)[-1])
        accepted[b], emitted[b, i], chances[b, i] = i, choice, p[choice]
    return dict(accepted=accepted, tokens=emitted, probabilities=chances)
