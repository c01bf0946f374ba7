"""What the entries over a paged cache refuse, before anything is launched: the
C ABI's status codes, and the Python wrappers' ValueErrors on host tensors."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
tq = pytest.importorskip("turboquant_amd")
lib = tq.lib

P = 0x1000  # an address that a refused call never reads
ALL = (1 << 64) - 1


def _plan(batch=2, width=4, cap=8, page=16, tokens=2, **null):
    a = dict(kv=P, new=P, table=P, free=P, count=P, slots=P, pos=P, starts=P, app=P, kvo=P, fo=P)
    a.update(null)
    return lib.tq_paged_plan(a["kv"], a["new"], batch, a["table"], width, a["free"], cap, a["count"], page, tokens,
                             a["slots"], a["pos"], a["starts"], a["app"], a["kvo"], a["fo"], None)


@pytest.mark.parametrize("kw", [dict(page=48), dict(page=8), dict(page=2048), dict(page=0), dict(batch=-1),
                                dict(batch=65536), dict(tokens=-1), dict(tokens=(1 << 24) + 1), dict(width=-1),
                                dict(width=(1 << 20) + 1), dict(cap=-1), dict(kv=None), dict(new=None),
                                dict(table=None), dict(free=None), dict(count=None), dict(slots=None), dict(pos=None),
                                dict(starts=None), dict(app=None), dict(kvo=None), dict(fo=None)])
def test_plan_refuses(kw):
    assert _plan(**kw) == 6
    assert lib.tq_last_error()


def _rope(dtype=1, tokens=3, heads=4, kv=2, d=64, rot=64, eps=1e-6, qs=None, ks=None, qos=None, kos=None, pos=P, q=P,
          inv=P):
    return lib.tq_qk_norm_rope(q, heads * d if qs is None else qs, P, kv * d if ks is None else ks, dtype, pos,
                               tokens, heads, kv, d, inv, rot, 0, None, None, eps, P,
                               heads * d if qos is None else qos, P, kv * d if kos is None else kos, None)


@pytest.mark.parametrize("kw,code", [(dict(dtype=3), 6), (dict(d=48, rot=32), 1), (dict(d=288), 1), (dict(rot=3), 1),
                                     (dict(rot=66), 1), (dict(rot=-2), 1), (dict(tokens=-1), 6), (dict(heads=-1), 6),
                                     (dict(eps=-1.0), 6), (dict(eps=float("nan")), 6), (dict(qs=255), 3),
                                     (dict(ks=127), 3), (dict(qos=255), 3), (dict(kos=0), 3), (dict(pos=None), 6),
                                     (dict(q=None), 6), (dict(inv=None), 6)])
def test_rope_refuses(kw, code):
    assert _rope(**kw) == code


def test_rope_of_nothing_is_nothing():
    assert _rope(tokens=0) == 0
    assert _rope(heads=0, kv=0) == 0


def _store(dtype=1, tokens=2, pages=4, heads=2, page=16, d=64, bits=3, ob=ALL, norm=0, stride=None, signs=None,
           norms=None, rm=None, slots=P, k=P, ki=0x1000, ks=0x1000):
    stride = heads * d if stride is None else stride
    return lib.tq_paged_store(k, stride, P, stride, dtype, slots, tokens, ki, ks, P, P, signs, norms, rm, pages, heads,
                              page, d, bits, ob, norm, None)


@pytest.mark.parametrize("kw,code", [(dict(page=17), 6), (dict(d=40), 6), (dict(heads=0), 6), (dict(heads=65536), 6),
                                     (dict(pages=-1), 6), (dict(pages=1 << 31), 6), (dict(bits=2), 2),
                                     (dict(bits=5), 2), (dict(norm=2), 6), (dict(ob=1), 6), (dict(dtype=7), 6),
                                     (dict(tokens=-1), 6), (dict(stride=127), 3), (dict(slots=None), 6),
                                     (dict(k=None), 6), (dict(ki=0x1004), 6), (dict(ks=0x1002), 6),
                                     (dict(signs=P, norms=P, rm=P), 6),                      # the outlier codebook
                                     (dict(signs=P, norms=P, rm=P, d=96, ob=0), 1),          # no sketch of 96
                                     (dict(signs=P, norms=None, rm=P, ob=0), 6),
                                     (dict(signs=P, norms=P, rm=None, ob=0), 6),
                                     (dict(tokens=1 << 30), 6)])
def test_store_refuses(kw, code):
    assert _store(**kw) == code


@pytest.mark.parametrize("call", ["store", "decode"])
@pytest.mark.parametrize("offset", [1, 4, 8])
def test_sign_pools_start_on_a_16_byte_boundary(call, offset):
    kw = dict(signs=0x1000 + offset, norms=P, rm=P, ob=0)
    assert (_store(**kw) if call == "store" else _decode(**kw)) == 6


def test_store_of_nothing_is_nothing():
    assert _store(tokens=0, k=None) == 0


def _load(tokens=2, pages=4, heads=2, page=16, d=64, bits=3, ob=ALL, dtype=0, slots=P, out=0x1000):
    return lib.tq_paged_load(P, P, P, P, slots, tokens, pages, heads, page, d, bits, ob, 0, out, P, dtype, None)


@pytest.mark.parametrize("kw,code", [(dict(page=0), 6), (dict(d=33), 6), (dict(bits=1), 2), (dict(dtype=-1), 6),
                                     (dict(tokens=-2), 6), (dict(slots=None), 6), (dict(out=0x1008), 6),
                                     (dict(ob=1), 6), (dict(tokens=1 << 30), 6)])
def test_load_refuses(kw, code):
    assert _load(**kw) == code


def _decode(qdt=1, odt=1, batch=2, heads=4, kv=2, d=64, bits=3, ob=ALL, norm=0, page=16, pages=8, width=4, most=64,
            signs=None, norms=None, rm=None, table=P, lens=P, ws=P, ws_bytes=1 << 30, q=P, ki=0x1000):
    return lib.tq_paged_decode_attention(q, qdt, ki, P, P, P, signs, norms, rm, table, width, lens, batch, heads, kv, d,
                                         bits, ob, norm, page, pages, most, 0.1, P, odt, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [(dict(page=24), 6), (dict(d=96), 6), (dict(bits=2), 2), (dict(ob=1), 6),
                                     (dict(heads=3), 6), (dict(heads=0), 6), (dict(qdt=5), 6), (dict(odt=5), 6),
                                     (dict(batch=-1), 6), (dict(batch=65536), 6), (dict(most=65), 6),
                                     (dict(most=-1), 6), (dict(width=-1), 6), (dict(table=None), 6),
                                     (dict(lens=None), 6), (dict(ws=None), 6), (dict(ws_bytes=256), 6),
                                     (dict(q=None), 6), (dict(signs=P, norms=P, rm=P), 6),
                                     (dict(signs=P, norms=P, rm=P, ob=0, d=32), 6),
                                     (dict(signs=P, norms=None, rm=P, ob=0), 6),
                                     (dict(signs=P, norms=P, rm=None, ob=0), 6)])
def test_decode_refuses(kw, code):
    assert _decode(**kw) == code


def test_decode_of_no_request_is_nothing():
    assert _decode(batch=0, q=None) == 0


# ---- the wrappers, on host tensors ----

def test_layer_shapes():
    k, s = torch.zeros((2, 1, 16, 24), dtype=torch.uint8), torch.zeros((2, 1, 16, 2), dtype=torch.int16)
    with pytest.raises(ValueError, match="current device"):
        tq.PagedLayer(k, s, k, s)
    with pytest.raises(ValueError, match="must be"):
        tq.PagedLayer(k.to(torch.int8), s, k, s)
    with pytest.raises(ValueError, match="pools"):
        tq.PagedLayer(k[0], s, k, s)


def test_plan_wrapper_shapes():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="current device"):
        tq.paged_plan(i(2), i(2), i(2, 3), i(4), i(1), 16, 2)
    with pytest.raises(ValueError, match="expected"):
        tq.paged_plan(i(2, 1), i(2), i(2, 3), i(4), i(1), 16, 2)
    with pytest.raises(ValueError, match="kv_lens must be"):
        tq.paged_plan(i(2).long(), i(2), i(2, 3), i(4), i(1), 16, 2)


def test_rope_wrapper_shapes():
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    pos, f = torch.zeros(3, dtype=torch.int32), torch.zeros(32)
    with pytest.raises(ValueError, match="current device"):
        tq.qk_norm_rope(q, k, pos, f, out=(q, k))
    with pytest.raises(ValueError, match="one type"):
        tq.qk_norm_rope(q, k.half(), pos, f)
    with pytest.raises(ValueError, match="one type"):
        tq.qk_norm_rope(q, k[:2], pos, f)


def test_cache_arguments():
    c = tq.CacheConfig(bits=3, head_dim=64, num_kv_heads=2, num_layers=1)
    for kw in (dict(page_size=24), dict(page_size=8), dict(num_pages=0), dict(max_requests=0), dict(max_kv_len=0),
               dict(qjl=True)):
        a = dict(num_pages=4, max_requests=2, max_kv_len=64)
        a.update(kw)
        with pytest.raises(ValueError):
            tq.PagedCache(c, device="cpu", **a)


def test_error_text_reaches_the_exception():
    with pytest.raises(tq.TurboQuantError, match="page_size 48"):
        from turboquant_amd._lib import check
        check(_plan(page=48))
    assert C.c_char_p(lib.tq_last_error()).value
