"""CPU: the paged-cache operators and the sampler refuse bad arguments before
touching a device."""
import ctypes

import pytest

vp = ctypes.c_void_p
F = vp(0x1000)  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib(ie):
    from infengine_b200 import paged
    paged._bind()
    return ie.lib()


def cache(**kw):
    from infengine_b200.paged import _Cache
    d = dict(k=0x1000, v=0x1000, num_pages=10, page_size=16, n_kv_heads=2, head_dim=128, page_stride=2 * 16 * 128,
             head_stride=16 * 128, row_stride=128)
    d.update(kw)
    return _Cache(**d)


CACHES = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(num_pages=0), -1), (dict(n_kv_heads=0), -1),
    (dict(head_dim=96), -3), (dict(head_dim=256), -3), (dict(page_size=8), -3), (dict(page_size=24), -3),
    (dict(page_size=512), -3), (dict(row_stride=64), -1), (dict(head_stride=64), -1), (dict(page_stride=64), -1),
    (dict(head_stride=15 * 128), -1),            # heads overlap
    (dict(page_stride=31 * 128), -1),            # pages overlap
    (dict(row_stride=132, head_stride=16 * 132, page_stride=32 * 132), -2),
    (dict(k=0x1008), -2), (dict(page_stride=1 << 37), -1),
]


@pytest.mark.parametrize("change,status", CACHES)
def test_cache_refusals(lib, change, status):
    assert attention(lib, cache=cache(**change)) == status
    assert norm(lib, cache=cache(**change)) == status


def attention(lib, **kw):
    a = dict(dt=1, B=2, T=4, max_q=2, heads=8, q=F, ldq=1024, hs=128, cache=cache(), table=F, ldt=8, pages=8, start=F,
             kv=F, window=0, sinks=0, scale=0.1, out=F, ldo=1024, ws=F, bytes=1 << 40)
    a.update(kw)
    c = a["cache"]
    return lib.ie_paged_attention(a["dt"], a["B"], a["T"], a["max_q"], a["heads"], a["q"], a["ldq"], a["hs"],
                                  ctypes.addressof(c) if c else None, a["table"], a["ldt"], a["pages"], a["start"],
                                  a["kv"], a["window"], a["sinks"], a["scale"], a["out"], a["ldo"], a["ws"],
                                  a["bytes"], None)


@pytest.mark.parametrize("change,status", [
    (dict(dt=2), -1), (dict(B=-1), -1), (dict(T=-1), -1), (dict(max_q=-1), -1), (dict(heads=0), -1),
    (dict(cache=None), -1), (dict(heads=9), -3), (dict(heads=34), -3), (dict(q=None), -1), (dict(out=None), -1),
    (dict(table=None), -1), (dict(start=None), -1), (dict(kv=None), -1), (dict(pages=0), -1), (dict(ldt=7), -1),
    (dict(pages=1 << 28, ldt=1 << 28), -1),      # positions past 32 bits
    (dict(pages=(1 << 27) - 8, ldt=1 << 28), -1),  # and those whose last block's end is
    (dict(window=-1), -1), (dict(sinks=-1), -1), (dict(sinks=4), -1),  # sinks without a window
    (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(hs=64), -1), (dict(ldq=-8), -1), (dict(ldo=1016), -1),
    (dict(q=vp(0x1008)), -2), (dict(out=vp(0x1002)), -2), (dict(ldq=1028), -2), (dict(hs=132), -2),
    (dict(ldo=1028), -2), (dict(ws=None), -7), (dict(bytes=1000), -7), (dict(ws=vp(0x1004)), -2),
    (dict(max_q=1 << 30, T=1 << 30), -3), (dict(table=vp(0x1002)), -2), (dict(start=vp(0x1001)), -2),
    (dict(kv=vp(0x1002)), -2),
    (dict(B=0), 0), (dict(T=0), 0), (dict(max_q=0), 0),
])
def test_attention_refusals(lib, change, status):
    assert attention(lib, **change) == status


def norm(lib, **kw):
    a = dict(dt=1, B=2, T=4, heads=8, q=F, ldq=1536, hq=128, k=F, ldk=1536, hk=128, v=F, ldv=1536, hv=128, qw=F, kw=F,
             eps=1e-5, cos=F, sin=F, rows=100, cache=cache(), table=F, ldt=8, pages=8, start=F, kv=F, out=F, ldo=1024,
             ho=128)
    a.update(kw)
    c = a["cache"]
    return lib.ie_qk_norm_rope_paged(a["dt"], a["B"], a["T"], a["heads"], a["q"], a["ldq"], a["hq"], a["k"], a["ldk"],
                                     a["hk"], a["v"], a["ldv"], a["hv"], a["qw"], a["kw"], a["eps"], a["cos"],
                                     a["sin"], a["rows"], ctypes.addressof(c) if c else None, a["table"], a["ldt"],
                                     a["pages"], a["start"], a["kv"], a["out"], a["ldo"], a["ho"], None)


@pytest.mark.parametrize("change,status", [
    (dict(dt=-1), -1), (dict(B=-1), -1), (dict(T=-1), -1), (dict(heads=0), -1), (dict(cache=None), -1),
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(table=None), -1),
    (dict(start=None), -1), (dict(kv=None), -1), (dict(cos=None), -1), (dict(sin=None), -1), (dict(rows=0), -1),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(hq=64), -1), (dict(ho=64), -1), (dict(ldo=8), -1),
    (dict(q=vp(0x1008)), -2), (dict(kw=vp(0x1008)), -2), (dict(cos=vp(0x1004)), -2), (dict(ldk=1540), -2),
    (dict(hv=130), -2), (dict(ldq=1 << 41), -1), (dict(ho=1 << 41), -1),
    (dict(ldo=7 * 128), -1), (dict(ldo=128, ho=3 * 128), -1), (dict(ldo=136, ho=3 * 136), -1),  # output rows overlap
    (dict(heads=70000, ldo=70000 * 128), -3), (dict(B=0), 0), (dict(T=0), 0),
])
def test_norm_rope_refusals(lib, change, status):
    assert norm(lib, **change) == status


@pytest.mark.parametrize("change,status", [
    (dict(dt=3), -1), (dict(M=-1), -1), (dict(V=-1, ld=0), -1), (dict(V=0), -1), (dict(ld=99), -1),
    (dict(x=None), -1), (dict(u=None), -1), (dict(idx=None), -1), (dict(x=vp(0x1001)), -2),
    (dict(u=vp(0x1002)), -2), (dict(idx=vp(0x1001)), -2),
    (dict(V=600000, ld=600000), -3), (dict(M=1 << 25), -3), (dict(M=0), 0),
])
def test_sample_refusals(lib, change, status):
    a = dict(dt=0, M=2, V=100, ld=100, x=F, u=F, idx=F)
    a.update(change)
    assert lib.ie_sample(a["dt"], a["M"], a["V"], a["x"], a["ld"], None, None, None, None, a["u"], a["idx"], None,
                         None) == status


def test_python_forms_refuse_cpu_tensors(ie):
    import torch
    x = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ie.PagedCache(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ie.sample(torch.zeros((1, 5), dtype=torch.float16), torch.zeros(1), torch.zeros(1, dtype=torch.int32))


def test_workspace_size(ie):
    n = ie.paged_attention_workspace_bytes()
    assert 0 < n < 64 << 20 and n == ie.lib().ie_paged_attention_workspace_size()
