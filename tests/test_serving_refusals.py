"""The serving operators refuse what they cannot compute, before any device work:
every call here is wrong on the host's side, so it is refused without a device."""
import ctypes as C

import pytest

import rustyneedle_amd as rn

lib = rn.lib
A = 1 << 20  # an address that is never followed


def cache(format=rn.CACHE_I8, sequences=2, kv_heads=2, capacity=16, keys=A, values=A, key_scales=A, value_scales=A,
          sequence_rows=None, head_rows=None):
    return rn.Cache.view(format, sequences, kv_heads, capacity, keys, values, key_scales, value_scales, sequence_rows,
                         head_rows).struct


def rows(type=rn.F32, keys=A, values=A, strides=(2048, 128, 64)):
    return rn.CacheRows(type, keys, values, *strides)


def refused(rc, *words):
    text = lib.rn_last_error().decode()
    assert rc == rn.RN_ERR_ARGUMENT, (rc, text)
    for w in words:
        assert w in text, text


@pytest.mark.parametrize("entry", ["rn_cache_write", "rn_cache_read"])
def test_cache_rows(entry):
    call = lambda c, r, tokens=4: getattr(lib, entry)(c, r, tokens, None, None, None, None)  # noqa: E731
    refused(call(None, rows()), "null")
    refused(call(cache(format=7), rows()), "format")
    for wrong in ("sequences", "kv_heads", "capacity"):
        refused(call(cache(**{wrong: 0}), rows()), "positive")
    refused(call(cache(sequences=65536, capacity=1), rows()), "65535")
    refused(call(cache(capacity=(1 << 24) + 1), rows()), "2^24")
    refused(call(cache(head_rows=15), rows()), "overlap")
    refused(call(cache(head_rows=16, sequence_rows=31), rows()), "overlap")
    refused(call(cache(head_rows=-16), rows()), "strides")
    refused(call(cache(key_scales=None), rows()), "scales")
    refused(call(cache(keys=None), rows()), "null")
    refused(call(cache(), None), "rows")
    refused(call(cache(), rows(keys=None)), "null")
    refused(call(cache(), rows(type=2)), "type")
    refused(call(cache(), rows(), -1), "tokens")
    refused(call(cache(), rows(), 17), "tokens")
    refused(call(cache(), rows(strides=(2048, 126, 64))), "16 bytes")
    refused(call(cache(), rows(type=rn.F16, strides=(2048, 132, 64))), "16 bytes")
    refused(call(cache(), rows(strides=(-2048, 128, 64))), "16 bytes")
    assert call(cache(), rows(), 0) == rn.RN_OK  # nothing to do


def test_rows_to_fill_may_not_overlap():
    read = lambda strides: lib.rn_cache_read(cache(), rows(strides=strides), 4, None, None, None, None)  # noqa: E731
    refused(read((512, 128, 32)), "overlap")
    refused(read((0, 128, 64)), "overlap")
    refused(read((256, 128, 64)), "overlap")  # the second sequence starts inside the first


def attend(prefix="i8", own="i8", sequences=2, queries=1, heads=4, prefix_length=8, lengths=A, counts=None, scale=0.125,
           window=0, workspace=A, workspace_bytes=1 << 30, q=A, out=A, q_stride=256, out_stride=256):
    made = {"i8": lambda n: cache(sequences=n), "f16": lambda n: cache(format=rn.CACHE_F16, sequences=n), None: lambda n: None}
    p = made[prefix](1) if not isinstance(prefix, rn.CacheView) else prefix
    o = made[own](2) if not isinstance(own, rn.CacheView) else own
    return lib.rn_attend_shared(q, q_stride, out, out_stride, sequences, queries, heads, p, prefix_length, o, lengths,
                                counts, scale, window, workspace, workspace_bytes, None, None)


def test_attend_shared():
    refused(attend(prefix=None, own=None, prefix_length=0), "neither")
    refused(attend(prefix=None), "without a prefix")
    refused(attend(own=None), "lengths")
    refused(attend(prefix_length=17), "prefix_length")
    refused(attend(prefix_length=-1), "prefix_length")
    refused(attend(sequences=3), "holds 2 sequences")
    refused(attend(sequences=-1), "shape")
    refused(attend(heads=3, q_stride=192, out_stride=192), "kv_heads")
    refused(attend(heads=130, q_stride=8320, out_stride=8320), "kv_heads")
    refused(attend(own=cache(kv_heads=4)), "differ")
    refused(attend(queries=65536), "2^20")
    refused(attend(queries=65535, sequences=2, heads=64, q_stride=4096, out_stride=4096), "2^20")
    for scale in (0.0, -1.0, 3e38, float("inf"), float("nan")):
        refused(attend(scale=scale), "scale")
    refused(attend(window=-1), "window")
    refused(attend(q=None), "null")
    refused(attend(out=None), "null")
    refused(attend(q_stride=255), "q_stride")
    refused(attend(out_stride=252), "q_stride")
    refused(attend(q_stride=258), "q_stride")
    long = cache(sequences=1, capacity=4096)  # (a short prefix needs no workspace)
    refused(attend(prefix=long, prefix_length=4000, workspace=None), "workspace")
    refused(attend(prefix=long, prefix_length=4000, workspace_bytes=64), "workspace")
    assert attend(sequences=0, q=None, out=None, workspace=None, workspace_bytes=0) == rn.RN_OK
    assert attend(queries=0, q=None, out=None, workspace=None, workspace_bytes=0) == rn.RN_OK


def test_attend_shared_workspace():
    size = C.c_size_t(1)
    assert lib.rn_attend_shared_workspace(0, 1, 4, cache(sequences=1), 8, cache(), C.byref(size)) == rn.RN_OK
    assert size.value == 0
    refused(lib.rn_attend_shared_workspace(2, 1, 4, cache(sequences=1), 8, cache(), None), "null")
    refused(lib.rn_attend_shared_workspace(2, 1, 3, cache(sequences=1), 8, cache(), C.byref(size)), "kv_heads")


def verify(sequences=2, drafts=3, vocab=100, target=A, target_stride=100, draft=A, draft_stride=100, tokens=A,
           uniforms=A, accepted=A, emitted=A, workspace=A, workspace_bytes=1 << 30):
    return lib.rn_verify_drafts(sequences, drafts, vocab, target, target_stride, draft, draft_stride, tokens, None,
                                None, uniforms, accepted, emitted, None, workspace, workspace_bytes, None, None)


def test_verify_drafts():
    refused(verify(sequences=-1), "sequences")
    refused(verify(sequences=65536), "sequences")
    refused(verify(drafts=64), "drafts")
    refused(verify(drafts=-1), "drafts")
    refused(verify(vocab=0), "vocab")
    refused(verify(vocab=(1 << 24) + 1), "vocab")
    for name in ("target", "tokens", "uniforms", "accepted", "emitted"):
        refused(verify(**{name: None}), "null")
    refused(verify(target_stride=99), "stride")
    refused(verify(draft_stride=99), "stride")
    refused(verify(workspace=None), "workspace")
    refused(verify(workspace_bytes=16), "workspace")
    assert verify(sequences=0, target=None) == rn.RN_OK
    size = C.c_size_t(0)
    refused(lib.rn_verify_drafts_workspace(2, 64, 100, C.byref(size)), "drafts")
    refused(lib.rn_verify_drafts_workspace(2, 3, 100, None), "null")


def test_layer_caches_refuse_nulls():
    out = rn.CacheView()
    for entry in ("rn_session_layer_cache", "rn_batch_layer_cache", "rn_n3_session_layer_cache"):
        refused(getattr(lib, entry)(None, 0, C.byref(out)), "null")


def test_a_cache_of_its_own_needs_a_size():
    with pytest.raises(ValueError):
        rn.Cache(rn.CACHE_I8, 1, 0, 16)
