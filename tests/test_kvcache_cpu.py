"""The key/value cache and the 4-bit layers without a GPU: what ops refuses before any device work, and what the C entry
points refuse before they look at their context."""
import ctypes

import pytest
import torch

import _kv
from sycl_minimax_h3_b200 import native, ops


def cache(dim=64, heads=2, seqs=3, weights=True, dtype=torch.float16, pages=5, width=4):
    return ops.KVCache.empty(pages, seqs, width, heads, dim, dtype, "cpu", weights)


def rows(T=4, heads=2, dim=64, dtype=torch.float16):
    return ops.Rows.packed(torch.zeros(T, heads * dim, dtype=dtype), heads, dim)


STARTS = torch.zeros(4, dtype=torch.int32)


def test_a_cache_checks_its_parts():
    c = cache()
    part = {n: getattr(c, n) for n in ("k", "v", "k_scale", "v_scale", "tail_k", "tail_v", "table", "lens", "weight", "tail_weight")}
    ops.KVCache(**part)
    for name, bad, why in (("k", c.k[:, :, :32], "64, dim"), ("v", c.v.float(), "v"), ("v", c.v.transpose(0, 1), "v"),
                           ("k_scale", c.k_scale[:4], "k_scale"), ("tail_v", c.tail_v.float(), "tail_v"),
                           ("tail_k", c.tail_k[:2].clone(), "tail_k"), ("table", c.table.long(), "table"), ("lens", c.lens[:2], "lens"),
                           ("weight", None, "together"), ("tail_weight", c.tail_weight[:, :, :3], "tail_weight")):
        with pytest.raises(native.H3Error, match=why):
            ops.KVCache(**{**part, name: bad})
    with pytest.raises(native.H3Error, match="64 or 128"):
        cache(dim=96)
    with pytest.raises(native.H3Error, match="float"):
        cache(dtype=torch.int32)


def test_append_refusals():
    c = cache()
    for k, v, starts, why in ((rows(), rows(5), STARTS, "same layout"), (rows(heads=1), rows(heads=1), STARTS, "heads"),
                              (rows(dtype=torch.float32), rows(dtype=torch.float32), STARTS, "cache has"),
                              (rows(), rows(), STARTS[:3], "starts"), (rows(), rows(), STARTS.long(), "starts"),
                              (rows(), rows(), STARTS, "on a GPU")):
        with pytest.raises(native.H3Error, match=why):
            ops.kv_append(c, k, v, starts)
    wide = ops.Rows(torch.zeros(4, 128, dtype=torch.float16), 1, 128, 4, 2, 64)
    with pytest.raises(native.H3Error, match="do not fit"):
        ops.kv_append(c, wide, wide, STARTS)


def test_attention_refusals():
    c, out = cache(), torch.zeros(4, 256, dtype=torch.float16)
    for q, cc, o, kw, why in ((rows(heads=3), c, out, {}, "query heads"), (rows(heads=4, dtype=torch.bfloat16), c, out, {}, "out"),
                              (rows(heads=4), c, out[:3], {}, "out"), (rows(heads=4), c, out.t().contiguous().t(), {}, "out"),
                              (rows(heads=4), cache(weights=False), out, {"accumulate": True}, "no weights"),
                              (rows(heads=4, dim=32), c, torch.zeros(4, 256, dtype=torch.float16), {}, "heads of 32"),
                              (rows(heads=4), c, out, {}, "on a GPU")):
        with pytest.raises(native.H3Error, match=why):
            ops.attention_cached(q, cc, STARTS, o, **kw)


def test_evict_refusals():
    c, spare = cache(), torch.zeros(3, 1, dtype=torch.int32)
    for cc, s, budget, kw, why in ((cache(weights=False), spare, 64, {}, "no weights"), (c, spare, 63, {}, "multiple"),
                                   (c, spare, 0, {}, "multiple"), (c, spare, 64, {"sinks": 4, "recent": 61}, "do not fit"),
                                   (c, spare, 64, {"sinks": -1, "recent": 0}, "do not fit"), (c, spare, 128, {}, "spare"),
                                   (c, spare, 64, {"recent": 8}, "on a GPU")):
        with pytest.raises(native.H3Error, match=why):
            ops.kv_evict(cc, s, budget, **kw)


def test_int4_refusals():
    tiles, scale = torch.zeros(2, 3, 128, dtype=torch.int32), torch.zeros(5, 20)
    lin = ops.Int4Linear(tiles, scale, 20, 150, 32)
    assert lin.inputs() == 150 and lin.outputs() == 20
    for args, why in (((tiles, scale, 20, 150, 16), "groups"), ((tiles[:1], scale, 20, 150, 32), "tiles"), ((tiles, scale[:4], 20, 150, 32), "scale"),
                      ((tiles, scale, 20, 150, 32, scale.half()), "zero"), ((tiles, scale, 20, 150, 32, None, torch.zeros(19)), "bias"),
                      ((tiles, scale.int(), 20, 150, 32), "float")):
        with pytest.raises(native.H3Error, match=why):
            ops.Int4Linear(*args)
    for x, out, why in ((torch.zeros(2, 149), torch.zeros(2, 20), "do not fit"), (torch.zeros(2, 150), torch.zeros(3, 20), "do not fit"),
                        (torch.zeros(150, 2).t(), torch.zeros(2, 20), "contiguous"), (torch.zeros(2, 150).int(), torch.zeros(2, 20), "float"),
                        (torch.zeros(2, 150), torch.zeros(2, 20), "on a GPU")):
        with pytest.raises(native.H3Error, match=why):
            lin.forward(x, out)
    with pytest.raises(native.H3Error, match="uint8"):
        ops.Int4Linear.pack(torch.zeros(4, 4), scale, 0)


# ---- the C entry points: with no context at all, so that a refusal that came too late would crash ----

def struct(**kw):
    c = cache()
    s = native.KVCacheStruct.from_buffer_copy(c._struct)
    for n, v in kw.items():
        setattr(s, n, v)
    return c, s


BAD_CACHES = [({"dt": 3}, "type"), ({"dim": 96}, "64 or 128"), ({"pages": -1}, "range"), ({"seqs": 0}, "range"), ({"heads": 0}, "range"),
              ({"width": 1 << 25}, "range"), ({"seqs": 1 << 20, "heads": 1 << 20}, "range"), ({"k": None}, "null"), ({"tail_v": None}, "null"),
              ({"table": None}, "null"), ({"lens": None}, "null"), ({"v": 8}, "16 bytes"), ({"weight": None}, "together")]


@pytest.mark.parametrize("kw,why", BAD_CACHES)
def test_c_refuses_a_bad_cache(kw, why):
    L = native.lib()
    keep, s = struct(**kw)
    for rc in (L.h3s_kv_append(None, ctypes.addressof(s), 16, 16, 4, 128, 16, 0),
               L.h3s_attention_cached(None, ctypes.addressof(s), 16, 4, 2, 128, 16, 0, 0, 16, 0, None, 0),
               L.h3s_kv_evict(None, ctypes.addressof(s), 16, 64, 0, 0, 16, 1 << 20)):
        assert rc == -1 and why in native.last_error()
    assert L.h3s_attention_cached_work(None, ctypes.addressof(s), 4, 2, 0, 0, 0) == 0


def test_c_refusals():
    L = native.lib()
    keep, s = struct()
    p = ctypes.addressof(s)
    nw = native.KVCacheStruct.from_buffer_copy(s)
    nw.weight = nw.tail_weight = None
    pn = ctypes.addressof(nw)
    assert L.h3s_kv_append(None, p, 16, 16, 0, 128, 16, 0) == 0                       # nothing to do
    assert L.h3s_attention_cached(None, p, 16, 0, 2, 128, 16, 0, 0, 16, 0, None, 0) == 0
    assert L.h3s_kv_evict(None, p, 16, 64 * 5, 0, 0, 16, 1 << 20) == 0                # longer than any sequence can be
    for rc, why in ((lambda: L.h3s_kv_append(None, None, 16, 16, 4, 128, 16, 0), "no cache"),
                    (lambda: L.h3s_kv_append(None, p, 16, 16, 4, 127, 16, 0), "stride"),
                    (lambda: L.h3s_kv_append(None, p, 16, None, 4, 128, 16, 0), "null"),
                    (lambda: L.h3s_kv_append(None, p, 16, 16, 1 << 31, 128, 16, 0), "too many"),
                    (lambda: L.h3s_attention_cached(None, p, 16, 4, 3, 192, 16, 0, 0, 16, 0, None, 0), "multiple"),
                    (lambda: L.h3s_attention_cached(None, p, 16, 4, 2, 127, 16, 0, 0, 16, 0, None, 0), "stride"),
                    (lambda: L.h3s_attention_cached(None, p, 16, 4, 2, 128, None, 0, 0, 16, 0, None, 0), "null"),
                    (lambda: L.h3s_attention_cached(None, pn, 16, 4, 2, 128, 16, 0, 0, 16, 1, None, 0), "no weights"),
                    (lambda: L.h3s_kv_evict(None, pn, 16, 64, 0, 0, 16, 1 << 20), "no weights"),
                    (lambda: L.h3s_kv_evict(None, p, 16, 65, 0, 0, 16, 1 << 20), "multiple"),
                    (lambda: L.h3s_kv_evict(None, p, 16, 64, 1, 64, 16, 1 << 20), "fit the budget"),
                    (lambda: L.h3s_kv_evict(None, p, None, 64, 0, 0, 16, 1 << 20), "null"),
                    (lambda: L.h3s_kv_evict(None, p, 16, 64, 0, 0, 16, 4 * 3 * 2 * 64 - 1), "work"),
                    (lambda: L.h3s_int4_linear(None, 16, 0, 1, 64, 16, 16, 16, None, 0, 48, None, 16, 0), "groups"),
                    (lambda: L.h3s_int4_linear(None, 16, 0, 1, 64, 24, 16, 16, None, 0, 32, None, 16, 0), "16 bytes"),
                    (lambda: L.h3s_int4_linear(None, 16, 0, 1, 64, 16, 16, None, None, 0, 32, None, 16, 0), "null"),
                    (lambda: L.h3s_int4_linear(None, 16, 5, 1, 64, 16, 16, 16, None, 0, 32, None, 16, 0), "type"),
                    (lambda: L.h3s_int4_pack(None, 16, 4, 63, 16), "even"), (lambda: L.h3s_int4_pack(None, None, 4, 64, 16), "null")):
        assert rc() == -1 and why in native.last_error(), native.last_error()
    for M, N, K in ((0, 16, 64), (1, 0, 64), (1, 16, 0)):
        assert L.h3s_int4_linear(None, 16, 0, M, K, 16, N, 16, None, 0, 32, None, 16, 0) == 0


def test_c_refuses_more_tiles_than_a_launch_has():
    L = native.lib()
    keep, s = struct(seqs=1 << 28, heads=5)
    p = ctypes.addressof(s)
    assert L.h3s_attention_cached(None, p, 16, 4, 5, 5 * 64, 16, 0, 0, 16, 0, None, 0) == -1 and "too many sequences" in native.last_error()
    assert L.h3s_attention_cached_work(None, p, 4, 5, 0, 0, 0) == 0


def test_the_definitions_of_the_tests():
    """quantised(): ties to even, infinities saturate, NaN is 0; a cache reads back what was put into its tail."""
    codes, scale = _kv.quantised(torch.tensor([[127.0, 0.5, 1.5, -2.5, float("inf"), float("nan")]]))
    assert codes.tolist() == [[127, 0, 2, -2, 127, 0]] and float(scale) == 1.0
    c = _kv.random_cache([70, 3], 2, 64, torch.float32, "cpu")
    assert _kv.sequence(c, 0, "k").shape == (70, 2, 64)
    assert torch.equal(_kv.sequence(c, 1, "v")[2, 1], c.tail_v[1, 1, 2].double())
    page = int(c.table[0, 0])
    assert torch.equal(_kv.sequence(c, 0, "k")[5, 1], c.k[page, 1, 5].double() * c.k_scale[page, 1].double())


@pytest.mark.parametrize("N", [(1 << 29) - 127, 1 << 29, (1 << 31) - 143, (1 << 31) - 17])
def test_c_refuses_outputs_that_an_int_cannot_count(N):
    """Up to the end of the last block of 128 outputs, and in bytes of float32 scales"""
    L = native.lib()
    for M in (1, 12, 40):
        assert L.h3s_int4_linear(None, 16, 0, M, 64, 16, N, 16, None, 0, 32, None, 16, 0) == -1 and "too large" in native.last_error()
    assert L.h3s_int4_pack(None, 16, N, 64, 16) == -1 and "too large" in native.last_error()
