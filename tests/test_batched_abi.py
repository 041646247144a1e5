"""The batched step's entry points without a GPU: arguments are refused before
a device is looked for, good ones report that there is none, and the workspace
is sized on the host."""
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


A = 1 << 20  # an address that nothing reads here


def cache(**kw):
    f = dict(keys=A, values=A, table=A, type=_lib.DN_BF16, pages=8, page_size=16, kv_heads=2, hd=64, sequences=3,
             table_stride=4, page_stride=2 * 16 * 64)
    f.update(kw)
    return _lib.PagedCache(**f)


def test_descriptors_match_the_header():
    """Field by field, in the header's order."""
    text = open(_lib.HEADER).read()
    for name, struct in (("dn_paged_cache", _lib.PagedCache), ("dn_logit_rules", _lib.LogitRules)):
        body = text[text.index("typedef struct " + name):text.index("} " + name)]
        plain = re.sub(r"/\*.*?\*/", "", body[body.index("{") + 1:], flags=re.S)
        names = [re.sub(r"[\s*]", "", part.split()[-1] if " " in part.strip() else part)
                 for line in plain.split(";") for part in line.split(",") if part.strip()]
        assert names == [n for n, _ in struct._fields_], name
        assert ctypes.sizeof(struct) == 8 * len(struct._fields_)


def test_workspace(L):
    need = L.dn_paged_attention_workspace
    small, more = need(cache(), 4, 3, 0, 64), need(cache(), 4, 300, 4096, 5000)
    assert 0 < small < more
    assert need(cache(), 4, 0, 0, 64) > 0
    assert need(cache(type=_lib.DN_F32), 4, 3, 0, 64) > 0
    for c, args, rc in [(cache(type=7), (4, 3, 0, 64), -1), (cache(hd=300), (4, 3, 0, 64), -5), (cache(), (5, 3, 0, 64), -1),
                        (cache(), (4, -3, 0, 64), -1), (cache(), (4, 3, -1, 64), -1), (None, (4, 3, 0, 64), -1)]:
        assert need(c, *args) == rc


@pytest.mark.skipif(has_gpu(), reason="checks the no-device behaviour")
def test_no_device(L):
    no = _lib.DN_ERR_NO_DEVICE
    need = L.dn_paged_attention_workspace(cache(), 4, 3, 16, 64)
    attend = lambda **kw: L.dn_paged_attention(*{**dict(c=cache(), q=A, qs=256, st=A, le=A, pp=A, pre=16, most=64, sc=1.0, w=0,
                                                        out=2 * A, os=256, h=4, n=3, ws=A, b=need, f=0, s=None), **kw}.values())
    assert attend() == no
    assert attend(b=need - 1) == -1 and attend(out=A + 2) == -1 and attend(h=3) == -1
    append = lambda **kw: L.dn_paged_append(*{**dict(c=cache(), t=2, q=A, qs=128, k=A, ks=128, v=A, vs=128, seq=A, pos=A, rope=A,
                                                     rows=64, rot=64, qn=None, kn=None, eps=1e-6, qo=2 * A, qos=128, h=2, n=5, f=0,
                                                     s=None), **kw}.values())
    assert append() == no
    assert append(rot=65) == -1 and append(ks=127) == -1 and append(qo=A + 2) == -1
    assert append(qo=A) == no  # in place: the same address, type and stride
    assert append(h=0, q=None, qo=None) == no and append(n=0) == 0
    apply = lambda **kw: L.dn_logits_apply(*{**dict(t=0, x=A, s=100, o=A, os=100, n=2, v=100, r=_lib.LogitRules(), f=0, st=None),
                                             **kw}.values())
    assert apply() == no
    assert apply(v=101) == -1 and apply(o=A + 4) == -1 and apply(r=None) == -1 and apply(n=0) == 0


def test_interleaved_rows_are_no_overlap(L):
    """q_out in the same wide rows as q, after it: equal byte strides, apart in every row."""
    args = dict(c=cache(), t=2, q=A, qs=512, k=A, ks=512, v=A, vs=512, seq=A, pos=A, rope=A, rows=64, rot=64, qn=None, kn=None,
                eps=1e-6, qo=A + 2 * 128, qos=512, h=2, n=5, f=0, s=None)
    if not has_gpu():
        assert L.dn_paged_append(*args.values()) == _lib.DN_ERR_NO_DEVICE
        args["qo"] = A + 2 * 127
        assert L.dn_paged_append(*args.values()) == _lib.DN_ERR_ARGS
        args["qo"] = A - 2 * 128 + 2 * 512  # the next row's q begins inside it
        assert L.dn_paged_append(*args.values()) == _lib.DN_ERR_NO_DEVICE
        args["qo"] += 2
        assert L.dn_paged_append(*args.values()) == _lib.DN_ERR_ARGS


def test_rotated_queries_apart_from_keys_and_values(L):
    """Rotated queries over keys or values that other threads still read are refused, as over other queries."""
    args = dict(c=cache(), t=2, q=A, qs=512, k=A + 2 * 128, ks=512, v=A + 2 * 256, vs=512, seq=A, pos=A, rope=A, rows=64, rot=64,
                qn=None, kn=None, eps=1e-6, qo=A, qos=512, h=2, n=5, f=0, s=None)
    call = lambda **kw: L.dn_paged_append(*{**args, **kw}.values())
    for kw in (dict(qo=A + 2 * 128), dict(qo=A + 2 * 256), dict(qo=A + 2 * 383), dict(qo=A + 2 * 4 * 512 + 2 * 300),
               dict(qo=A + 2 * 256, qos=256), dict(q=A + 2 * 384, qo=A + 2 * 129)):
        assert call(**kw) == _lib.DN_ERR_ARGS, kw
    if not has_gpu():
        assert call() == _lib.DN_ERR_NO_DEVICE  # in place, beside its keys and values
        assert call(qo=A + 2 * 384) == _lib.DN_ERR_NO_DEVICE  # after them in the same rows
        assert call(h=0, q=None, qo=None) == _lib.DN_ERR_NO_DEVICE
