"""The 8-bit cache's, the residual norm's and the sampler's entry points without
a GPU: arguments are refused before a device is looked for, good ones report
that there is none, descriptors match the header."""
import ctypes
import os
import re

import pytest

import dianoia_b200
from dianoia_b200 import _lib


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(dianoia_b200.LIB_PATH):
        from dianoia_b200 import build
        build.build()
    return dianoia_b200.lib()


def has_gpu():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


A, MB = 1 << 30, 1 << 20  # an address that nothing reads here
ARGS, LARGE, NONE = _lib.DN_ERR_ARGS, _lib.DN_ERR_TOO_LARGE, _lib.DN_ERR_NO_DEVICE


def cache(**kw):
    f = dict(keys=A, values=A + MB, key_scales=A + 2 * MB, value_scales=A + 3 * MB, table=A + 4 * MB, pages=8, page_size=16,
             kv_heads=2, hd=64, sequences=3, table_stride=4, page_stride=2 * 16 * 64, scale_stride=2 * 16)
    f.update(kw)
    return _lib.PagedQ8Cache(**f)


BAD_CACHES = [(None, ARGS), (cache(hd=8), ARGS), (cache(hd=72), ARGS), (cache(hd=272, page_stride=1 << 16), LARGE), (cache(pages=-1), ARGS),
              (cache(page_size=0), ARGS), (cache(kv_heads=0), ARGS), (cache(page_stride=2 * 16 * 64 - 16), ARGS),
              (cache(page_stride=2 * 16 * 64 + 8), ARGS), (cache(scale_stride=31), ARGS), (cache(keys=A + 8), ARGS),
              (cache(values=None), ARGS), (cache(key_scales=A + 2), ARGS), (cache(table=None), ARGS), (cache(table=A + 2), ARGS),
              (cache(page_size=1 << 20, table_stride=1 << 20, page_stride=1 << 32, scale_stride=1 << 32), LARGE)]


def test_descriptors_match_the_header():
    text = open(_lib.HEADER).read()
    for name, struct in (("dn_paged_q8_cache", _lib.PagedQ8Cache), ("dn_sampling", _lib.Sampling)):
        body = text[text.index("typedef struct " + name):text.index("} " + name)]
        plain = re.sub(r"/\*.*?\*/", "", body[body.index("{") + 1:], flags=re.S)
        names = [re.sub(r"[\s*]", "", part.split()[-1] if " " in part.strip() else part)
                 for line in plain.split(";") for part in line.split(",") if part.strip()]
        assert names == [n for n, _ in struct._fields_], name
        assert ctypes.sizeof(struct) == 8 * len(struct._fields_)


def refuses(call, bad):
    """Each of `bad` (keywords, code) is refused; the call as it stands finds no device."""
    if not has_gpu():
        assert call() == NONE
    for kw, rc in bad:
        assert call(**kw) == rc, kw


def test_append(L):
    X = 2 * A
    args = dict(c=cache(), t=2, q=X, qs=512, k=X + 2 * 128, ks=512, v=X + 2 * 256, vs=512, seq=A, pos=A, rope=A, rows=64, rot=64,
                qn=None, kn=None, eps=1e-6, ot=2, qo=X + MB, qos=128, h=2, n=5, f=0, s=None)
    call = lambda **kw: L.dn_paged_q8_append(*{**args, **kw}.values())
    refuses(call, [(dict(c=c), rc) for c, rc in BAD_CACHES] + [
        (dict(t=3), ARGS), (dict(ot=-1), ARGS), (dict(n=-1), ARGS), (dict(h=-1), ARGS), (dict(rot=65), ARGS), (dict(rot=-2), ARGS),
        (dict(rot=66), ARGS), (dict(rows=-1), ARGS), (dict(ks=127), ARGS), (dict(vs=127), ARGS), (dict(qs=127), ARGS),
        (dict(qos=127), ARGS), (dict(qs=(1 << 32) + 1), LARGE), (dict(n=1 << 30), LARGE), (dict(h=1 << 21, qs=1 << 31, qos=1 << 31), LARGE),
        (dict(k=None), ARGS), (dict(v=None), ARGS), (dict(q=None), ARGS), (dict(qo=None), ARGS), (dict(seq=None), ARGS),
        (dict(rope=None), ARGS), (dict(pos=A + 2), ARGS), (dict(k=X + 1), ARGS), (dict(ot=0, qo=X + MB + 2), ARGS),
        (dict(qo=X + 2 * 127, qos=512), ARGS), (dict(qo=X + 2 * 130, qos=512), ARGS), (dict(qo=X + 2 * 300, qos=512), ARGS),
        (dict(qo=A), ARGS), (dict(k=A + MB + 64), ARGS), (dict(v=A + 2 * MB), ARGS), (dict(q=A + 3 * MB), ARGS)])
    assert call(n=0) == 0
    if not has_gpu():
        for kw in (dict(qo=X, qos=512), dict(h=0, q=None, qo=None), dict(rot=0, rope=None), dict(qo=X + 2 * 384, qos=512)):
            assert call(**kw) == NONE, kw


def test_read(L):
    X = 2 * A
    args = dict(c=cache(), t=2, seq=A, pos=A, k=X, ks=128, v=X + MB, vs=128, n=5, f=0, s=None)
    call = lambda **kw: L.dn_paged_q8_read(*{**args, **kw}.values())
    refuses(call, [(dict(c=c), rc) for c, rc in BAD_CACHES] + [
        (dict(t=5), ARGS), (dict(n=-1), ARGS), (dict(ks=127), ARGS), (dict(vs=127), ARGS), (dict(seq=None), ARGS), (dict(pos=A + 1), ARGS),
        (dict(k=X + 1), ARGS), (dict(v=X + 200), ARGS), (dict(k=A + 64), ARGS), (dict(v=A + 3 * MB), ARGS), (dict(n=1 << 30), LARGE),
        (dict(vs=1 << 33), LARGE)])
    assert call(n=0) == 0 and call(k=None, v=None) == 0
    if not has_gpu():
        for kw in (dict(k=None, ks=0), dict(v=None, vs=0), dict(k=X, ks=256, v=X + 256, vs=256)):
            assert call(**kw) == NONE, kw


def test_attention(L):
    X = 2 * A
    need = L.dn_paged_q8_attention_workspace
    assert 0 < need(cache(), 4, 3, 64) and need(cache(), 4, 0, 0) > 0
    for c, rc in BAD_CACHES:
        assert need(c, 4, 3, 64) == rc
    assert need(cache(), 3, 3, 64) == ARGS and need(cache(), 4, -1, 64) == ARGS and need(cache(), 4, 3, -1) == ARGS
    assert need(cache(), 0, 3, 64) == ARGS and need(cache(), 4, 1 << 25, 64) == LARGE and need(cache(), 4, 3, 1 << 31) == LARGE
    bytes_ = need(cache(), 4, 3, 64)
    args = dict(c=cache(), t=2, q=X, qs=256, st=A, le=A, most=64, sc=1.0, w=0, out=X + MB, os=256, h=4, n=3, ws=X + 2 * MB, b=bytes_,
                f=0, s=None)
    call = lambda **kw: L.dn_paged_q8_attention(*{**args, **kw}.values())
    refuses(call, [(dict(c=c), rc) for c, rc in BAD_CACHES] + [
        (dict(t=3), ARGS), (dict(h=3), ARGS), (dict(w=-1), ARGS), (dict(w=1 << 31), ARGS), (dict(qs=255), ARGS), (dict(os=255), ARGS),
        (dict(b=bytes_ - 1), ARGS), (dict(ws=X + 2 * MB + 8), ARGS), (dict(ws=None), ARGS), (dict(q=None), ARGS), (dict(out=None), ARGS),
        (dict(le=None), ARGS), (dict(le=A + 2), ARGS), (dict(out=X + 1), ARGS), (dict(out=X + 2), ARGS), (dict(out=A + 64), ARGS),
        (dict(ws=X), ARGS), (dict(st=None, n=2), ARGS), (dict(os=(1 << 32) + 1), LARGE)])
    assert call(n=0) == 0
    if not has_gpu():
        assert call(out=X) == NONE and call(st=None) == NONE


def test_residual_norm(L):
    X = 2 * A
    args = dict(t=2, y=X, ys=64, post=A, g=X + MB, gs=64, sc=1.0, xt=0, x=X + 2 * MB, xs=64, xo=X + 3 * MB, xos=64, pre=A + MB, eps=1e-6,
                h=X + 4 * MB, hs=64, qa=X + 5 * MB, qas=72, rows=5, cols=64, f=0, s=None)
    call = lambda **kw: L.dn_residual_norm(*{**args, **kw}.values())
    refuses(call, [
        (dict(t=3), ARGS), (dict(xt=-1), ARGS), (dict(rows=-1), ARGS), (dict(cols=-1), ARGS), (dict(ys=63), ARGS), (dict(gs=63), ARGS),
        (dict(xs=63), ARGS), (dict(xos=63), ARGS), (dict(hs=63), ARGS), (dict(qas=71), ARGS), (dict(qas=74), ARGS), (dict(qa=X + 5 * MB + 2), ARGS),
        (dict(cols=48), ARGS), (dict(pre=None), ARGS), (dict(pre=None, h=None), ARGS), (dict(y=None), ARGS), (dict(x=None), ARGS),
        (dict(xo=None), ARGS), (dict(y=X + 1), ARGS), (dict(x=X + 2 * MB + 2), ARGS), (dict(post=A + 2), ARGS),
        (dict(cols=32769, ys=1 << 16, gs=1 << 16, xs=1 << 16, xos=1 << 16, hs=1 << 16), LARGE), (dict(rows=1 << 31), LARGE),
        (dict(xo=X + 2 * MB + 4), ARGS), (dict(xo=X + 2 * MB, xos=65), ARGS), (dict(h=X + 2), ARGS), (dict(h=X + MB), ARGS),
        (dict(h=X + 3 * MB), ARGS), (dict(qa=X + 3 * MB), ARGS), (dict(qa=X + 4 * MB), ARGS), (dict(xo=A), ARGS), (dict(h=A + MB), ARGS),
        (dict(g=X + 4 * MB + 64, gs=0), ARGS)])
    assert call(rows=0) == 0 and call(cols=0) == 0
    if not has_gpu():
        for kw in (dict(xo=X + 2 * MB), dict(h=X), dict(post=None, g=None, gs=0), dict(h=None, hs=0), dict(qa=None, qas=0, cols=63),
                   dict(pre=None, h=None, qa=None), dict(gs=0)):
            assert call(**kw) == NONE, kw


def test_sample(L):
    how = lambda **kw: _lib.Sampling(**{**dict(temperature=A, top_k=A + 64, top_p=A + 128, min_p=A + 192, uniform=A + 256), **kw})
    X = 2 * A
    args = dict(t=0, x=X, st=100, n=4, v=100, how=how(), tok=A + MB, lp=A + MB + 64, ke=A + MB + 128, f=0, s=None)
    call = lambda **kw: L.dn_sample(*{**args, **kw}.values())
    refuses(call, [
        (dict(t=4), ARGS), (dict(n=-1), ARGS), (dict(v=-1), ARGS), (dict(v=101), ARGS), (dict(how=None), ARGS), (dict(how=how(uniform=None)), ARGS),
        (dict(how=how(top_k=A + 2)), ARGS), (dict(tok=None), ARGS), (dict(x=None), ARGS), (dict(x=X + 2), ARGS), (dict(tok=A + MB + 1), ARGS),
        (dict(v=(1 << 19) + 1, st=1 << 20), LARGE), (dict(st=(1 << 32) + 1), LARGE), (dict(n=(1 << 24) + 1), LARGE), (dict(lp=A + MB + 8), ARGS),
        (dict(ke=X + 1200), ARGS), (dict(tok=A + 256), ARGS)])
    assert call(n=0) == 0
    if not has_gpu():
        for kw in (dict(lp=None, ke=None), dict(how=how(temperature=None, top_k=None, top_p=None, min_p=None)), dict(v=0, x=None, st=0), dict(t=2, x=X + 2)):
            assert call(**kw) == NONE, kw
