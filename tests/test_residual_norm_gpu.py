"""dn_residual_norm against its definition in 64 bits (tests/paged_q8_reference.py
derives the bounds): types, widths from one to the largest, strides and
alignments, every part on and off, outputs in place, QA blocks, graphs."""
import ctypes

import pytest

from tests import paged_q8_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from dianoia_b200 import _lib  # noqa: E402

TYPES = ref.TYPES


def stream():
    return torch.cuda.current_stream().cuda_stream


class Case:
    def __init__(self, kind, x_kind, rows, cols, post=True, gate="none", scale=1.0, pre=True, pad=0, offset=0, seed=0, qa=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dt, xdt = TYPES[kind][0], TYPES[x_kind][0]
        self.kind, self.x_kind, self.rows, self.cols, self.scale = kind, x_kind, rows, cols, scale

        def make(dtype, n=rows, size=3.0, fill=None):
            raw = torch.full((n * (cols + pad) + offset,), 7.0, device="cuda", dtype=dtype)
            part = raw[offset:].view(n, cols + pad)[:, :cols]
            if fill is None:
                part.copy_(torch.randn((n, cols), generator=g, device="cuda") * size)
            return part
        self.y, self.x = make(dt), make(xdt, size=2.0)
        self.gate = None if gate == "none" else make(dt, rows if gate == "each" else 1, 1.0)
        self.gate_stride = cols + pad if gate == "each" else 0
        vec = lambda: (1 + 0.2 * torch.randn(cols + offset, generator=g, device="cuda"))[offset:]
        self.post, self.pre = vec() if post else None, vec() if pre else None
        self.x_out, self.h = make(xdt, fill=7), make(dt, fill=7) if pre else None
        self.qa = torch.full((rows, cols // 32 * 36 + 8), 7, dtype=torch.uint8, device="cuda") if qa else None

    def call(self, L, flags=0, s=None):
        ptr = lambda t: None if t is None else t.data_ptr()
        step = lambda t: 0 if t is None else t.stride(0)
        return L.dn_residual_norm(TYPES[self.kind][1], ptr(self.y), step(self.y), ptr(self.post), ptr(self.gate), self.gate_stride,
                                  self.scale, TYPES[self.x_kind][1], ptr(self.x), step(self.x), ptr(self.x_out), step(self.x_out),
                                  ptr(self.pre), 1e-5, ptr(self.h), step(self.h), ptr(self.qa), step(self.qa), self.rows, self.cols,
                                  flags, stream() if s is None else s)

    def want(self):
        return ref.residual_norm(self.kind, self.x_kind, self.y, self.post, self.gate, self.scale, self.x, self.pre, 1e-5)

    def check(self, L, **kw):
        x, x_tol, h, h_tol = self.want()
        assert self.call(L, **kw) == 0
        torch.cuda.synchronize()
        assert ((self.x_out.double() - x).abs() <= x_tol).all()
        if self.h is not None:
            off = (self.h.double() - h).abs()
            assert (off <= h_tol).all(), float((off / h_tol).max())
        return self


KINDS = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"), ("f32", "bf16")]


@pytest.mark.parametrize("kind,x_kind", KINDS)
@pytest.mark.parametrize("cols", [1, 2, 31, 33, 100, 1000, 1024, 2048, 2050, 4096, 5120, 8192, 12288, 20000, 32767, 32768])
def test_widths(cuda_lib, kind, x_kind, cols):
    for rows, gate in ((1, "each"), (5, "one")):
        Case(kind, x_kind, rows, cols, gate=gate, scale=0.3, seed=cols).check(cuda_lib)


@pytest.mark.parametrize("kind,x_kind", KINDS)
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate", ["none", "one", "each"])
@pytest.mark.parametrize("pre", [True, False])
def test_parts(cuda_lib, kind, x_kind, post, gate, pre):
    for cols, pad, offset in ((256, 0, 0), (256, 8, 0), (256, 1, 0), (256, 0, 1), (77, 3, 0)):
        c = Case(kind, x_kind, 7, cols, post, gate, -0.5, pre, pad, offset).check(cuda_lib)
        if pad:
            base = c.x_out._base
            assert (base[offset:].view(7, cols + pad)[:, cols:] == 7).all()


@pytest.mark.parametrize("rows", [1, 2, 147, 148, 149, 1000, 5003])
def test_rows(cuda_lib, rows):
    for kind, x_kind, cols in (("bf16", "f32", 512), ("f32", "f32", 72), ("f16", "f16", 2048)):
        Case(kind, x_kind, rows, cols, gate="each", seed=rows).check(cuda_lib)


def test_in_place(cuda_lib):
    for kind in TYPES:
        for cols, pad in ((2048, 0), (333, 2)):
            c = Case(kind, kind, 9, cols, gate="one", pad=pad)
            x, x_tol, h, h_tol = c.want()
            c.x_out, c.h = c.x, c.y
            assert c.call(cuda_lib) == 0
            assert ((c.x.double() - x).abs() <= x_tol).all() and ((c.y.double() - h).abs() <= h_tol).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cols,pad", [(32, 0), (96, 0), (2048, 0), (6144, 0), (256, 1), (8192, 0), (32768, 0), (1056, 0)])
def test_qa_blocks(cuda_lib, kind, cols, pad):
    """In f32 the blocks are what dn_quantize_qa makes of h, bit for bit; h may be left out."""
    c = Case(kind, "f32", 6, cols, gate="each", pad=pad, qa=True).check(cuda_lib)
    blocks = cols // 32 * 36
    assert (c.qa[:, blocks:] == 7).all()
    got = c.qa[:, :blocks].clone()
    if kind == "f32":
        h = c.h.contiguous()
        want = torch.zeros((6, blocks), dtype=torch.uint8, device="cuda")
        assert cuda_lib.dn_quantize_qa(h.data_ptr(), want.data_ptr(), 6, cols, blocks, stream()) == 0
        assert torch.equal(got, want)
    else:  # from the f32 h: half a step, and h's own rounding
        b = got.view(6, cols // 32, 36).contiguous()
        scale = b[..., 32:].contiguous().view(torch.float32)
        value = (b[..., :32].view(torch.int8).double() * scale.double()).view(6, cols)
        _, _, h, h_tol = c.want()
        step = scale.double().expand(-1, -1, 32).reshape(6, cols)
        assert ((value - h).abs() <= step * 0.5001 + h_tol).all()
    c.h = None
    c.qa.fill_(7)
    assert c.call(cuda_lib) == 0
    assert torch.equal(c.qa[:, :blocks], got)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cols", [2056, 2080, 3000, 4064, 4088, 4104, 4128, 8160, 8200, 16384, 16416])
def test_runs_that_do_not_fill_the_threads(cuda_lib, kind, cols):
    """Rows in runs of 8 values on either side of each number of runs a thread, with QA blocks where a row is whole blocks."""
    if cols % 32 == 0:
        test_qa_blocks(cuda_lib, kind, cols, 0)
    Case(kind, "f32", 300, cols, gate="one", seed=cols).check(cuda_lib)


def test_values_of_every_size(cuda_lib):
    c = Case("f32", "f32", 4, 256)
    c.y[0], c.y[1] = 0, c.y[1] * 1e15
    c.x[0], c.x[2] = 0, c.x[2] * 1e-20
    c.check(cuda_lib)
    c.y[3, 5] = float("nan")
    assert c.call(cuda_lib) == 0
    assert c.h[3].isnan().all() and c.h[:3].isfinite().all()


def test_graph_and_stream(cuda_lib):
    c = Case("bf16", "f32", 33, 2048, gate="one")
    want = c.check(cuda_lib).h.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            assert c.call(cuda_lib, flags=_lib.DN_FLAG_PDL) == 0
    c.h.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.h, want)
    c.h.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert c.call(cuda_lib, s=s.cuda_stream) == 0
    s.synchronize()
    assert torch.equal(c.h, want)


def test_far_rows(cuda_lib):
    """Rows past 2^32 bytes."""
    rows, cols, pad = 3, 64, (1 << 30) - 64 + 8
    x = torch.zeros(2 * (cols + pad) + cols, device="cuda", dtype=torch.float32)
    y = torch.randn((rows, cols), device="cuda")
    view = torch.as_strided(x, (rows, cols), (cols + pad, 1))
    view.copy_(torch.randn((rows, cols), device="cuda"))
    want, tol, _, _ = ref.residual_norm("f32", "f32", y, None, None, 1.0, view, None, 1e-5)
    assert cuda_lib.dn_residual_norm(0, y.data_ptr(), cols, None, None, 0, 1.0, 0, x.data_ptr(), cols + pad, x.data_ptr(), cols + pad,
                                     None, 1e-5, None, 0, None, 0, rows, cols, 0, stream()) == 0
    assert ((view.double() - want).abs() <= tol).all()
