"""nls_g4_matmul: 4-bit weights with group scales, against the definition in
64 bits.

Tolerance. With q' = q - 8 the kernel computes s * sum(q' x) + m' * sum(x),
m' = m + 8 s, per group. More than 12 batch rows (4 with groups of 32):
products of a 4-bit and a 16-bit (or a third of an fp32) value are exact in
fp32, and every other operation rounds to fp32 or, in the tensor core's
accumulator, cuts off, so is off by at most 2^-23 relative to the sum of
magnitudes so far. Fewer rows: the inner sums are exact but for each x, which is
off by 2^-31 of the largest of its 128 columns; where activations are of one
size that is far below 2^-23 of the sum (a test of its own has one that is not). A logit is a sum of at most `group` terms,
then of the groups' terms, with fewer than 8 further roundings (m', its sum,
the scalings, the parts of a split tile), so it is within
(group + 3 * groups + 8) * 2^-23 * A of the exact value, A the same sum of
magnitudes; then it is rounded once to the output type (half a step: eps / 2).
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

DTYPES = ("f32", "f16", "bf16")


def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def make(pkg, rows, cols, group, stype="f16", mins=False, seed=0, device="cuda"):
    import torch
    g = torch.Generator().manual_seed(seed)
    groups = -(-cols // group)
    v = torch.randint(0, 16, (rows, cols), generator=g, dtype=torch.uint8)
    s = (0.5 + torch.rand((rows, groups), generator=g)) * 0.02
    s *= torch.where(torch.rand((rows, groups), generator=g) < 0.3, -1.0, 1.0)
    m = (-s * (8 + torch.rand((rows, groups), generator=g))).to(_dt(stype)).to(device) if mins else None
    return pkg.g4_pack(v.to(device), s.to(_dt(stype)).to(device), m, group=group)


def parts(w):
    """(w as float64 [rows, cols], magnitudes of the terms the kernel adds)."""
    import torch
    q = torch.stack((w.q & 15, w.q >> 4), 2).reshape(w.rows, w.cols).double()
    wide = lambda t: t.t().double().repeat_interleave(w.group, 1)[:, :w.cols]  # noqa: E731
    s = wide(w.scales)
    if w.mins is None:
        return (q - 8) * s, ((q - 8) * s).abs()
    m = wide(w.mins)
    return q * s + m, ((q - 8) * s).abs() + (m + 8 * s).abs()


def check(w, x, y, what=""):
    import torch
    W, A = parts(w)
    xd = x.double().reshape(-1, w.cols)
    want, mag = xd @ W.t(), xd.abs() @ A.t()
    groups = -(-w.cols // w.group)
    info = torch.finfo(y.dtype)
    tol = (min(w.group, w.cols) + 3 * groups + 8) * 2.0 ** -23 * mag
    tol = tol + (want.abs() + tol) * info.eps / 2 + info.smallest_normal * info.eps
    err = (y.double().reshape(want.shape) - want).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max())} of the tolerance"


# ---- host side ------------------------------------------------------------------

def test_pack_and_quantize_on_the_host(pkg):
    import torch
    g = torch.Generator().manual_seed(3)
    v = torch.randint(0, 16, (37, 96), generator=g)
    s = torch.rand((37, 3), generator=g)
    w = pkg.g4_pack(v, s, group=32)
    assert w.q.shape == (37, 48) and w.q.stride(0) % 16 == 0 and w.struct.s_ld == 40
    assert torch.equal(w.dequantize(), (v.float() - 8) * s.repeat_interleave(32, 1))
    wt = torch.randn((33, 160), generator=g)
    for group, sym in ((32, True), (64, False), (128, True), (256, False)):
        w = pkg.g4_quantize(wt, group, symmetric=sym)
        step = w.scales.t().abs().repeat_interleave(group, 1)[:, :160]
        d = (w.dequantize() - wt).abs()
        # to the nearest of 16 steps; symmetric levels stop at +7 steps, so a
        # value of the other sign near 8 steps is up to one step off
        assert bool((d <= step * (1.0 if sym else 0.5) + 1e-5).all())
    z = pkg.g4_quantize(torch.zeros((4, 64)), 32)
    assert not z.dequantize().any()


def test_host_refusals(pkg):
    import torch
    v, s = torch.zeros((16, 64), dtype=torch.uint8), torch.ones((16, 2))
    with pytest.raises(ValueError):
        pkg.g4_pack(v + 16, s, group=32)
    with pytest.raises(ValueError):
        pkg.g4_pack(v[:, :48], s, group=32)               # columns not in whole 32
    with pytest.raises(ValueError):
        pkg.g4_pack(v, s, group=48)
    with pytest.raises(ValueError):
        pkg.g4_pack(v, s, group=64)                       # one group per row, two given
    with pytest.raises(TypeError):
        pkg.g4_pack(v, s.double(), group=32)
    w = pkg.g4_pack(v, s, group=32)
    with pytest.raises(ValueError):                       # mins of another type
        pkg.G4Weights(w.q, w.scales, w.scales.half(), group=32)
    with pytest.raises(ValueError):                       # no room behind the last line
        pkg.G4Weights(torch.zeros((20, 16), dtype=torch.uint8), torch.ones((1, 20)), group=32)
    lib = pkg.load()
    assert lib.nls_g4_matmul(None, ctypes.byref(w.struct), None, 0, 64, 1, None, 0, 16, 0, None) == 1
    assert lib.nls_g4_lm_head_draw(None, ctypes.byref(w.struct), None, 0, 64, 1, 0, None, None, None, None, 0, None) == 1


def test_struct_layout_matches_c(pkg, tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in pkg._abi.G4WeightsStruct._fields_]
    dn = list(pkg.DRAW_PARAMS_DTYPE.names)
    prog = "#include <stdio.h>\n#include <stddef.h>\n#include \"nimllm_sample.h\"\nint main(void) {\n" + \
        "printf(\"%zu %zu\\n\", sizeof(nls_g4_weights), sizeof(nls_draw_params));\n" + \
        "".join(f'printf("%zu\\n", offsetof(nls_g4_weights, {n}));\n' for n in names) + \
        "".join(f'printf("%zu\\n", offsetof(nls_draw_params, {n}));\n' for n in dn) + "return 0; }\n"
    c = tmp_path / "t.c"
    c.write_text(prog)
    exe = str(tmp_path / "t")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(c), "-o", exe], check=True)
    vals = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert vals[:2] == [ctypes.sizeof(pkg._abi.G4WeightsStruct), pkg.DRAW_PARAMS_DTYPE.itemsize]
    assert vals[2:2 + len(names)] == [getattr(pkg._abi.G4WeightsStruct, n).offset for n in names]
    assert vals[2 + len(names):] == [pkg.DRAW_PARAMS_DTYPE.fields[n][1] for n in dn]


def test_a_failed_host_call_raises_with_check_off(pkg):
    """check=False does not wait for a device call's kernels; a host call has
    waited, and its result is not handed out when it has failed."""
    import types
    import torch
    w = types.SimpleNamespace(device=torch.device("cuda", 0), struct=pkg._abi.G4WeightsStruct(), rows=16, cols=64)

    class Lib:
        status = 0

        def nls_g4_matmul(self, *args):
            return self.status

        def nls_last_error(self, h):
            return b""

        def nls_destroy(self, h):
            pass

    eng = pkg.Engine.__new__(pkg.Engine)
    eng._lib, eng._h, eng.device, eng._torch_device = Lib(), None, 0, None
    x = torch.zeros((2, 64))
    for check in (True, False):
        Lib.status = 0
        assert eng.g4_matmul(w, x, check=check).shape == (2, 16)
        for status in (pkg._abi.NLS_ERR_TIMEOUT, pkg._abi.NLS_ERR_CUDA, pkg._abi.NLS_ERR_INVALID_ARG):
            Lib.status = status
            with pytest.raises(pkg.NlsError) as e:
                eng.g4_matmul(w, x, check=check)
            assert e.value.status == status


# ---- GPU ------------------------------------------------------------------------

@pytest.fixture(scope="module")
def eng(pkg):
    e = pkg.Engine(0, max_rows=64, max_vocab=1 << 17)
    yield e
    e.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,group,mins,nb", [
    (1, 32, 32, False, 1),            # the smallest
    (7, 64, 128, True, 3),            # one short group
    (128, 128, 128, False, 1),        # one tile, one step
    (129, 160, 32, True, 2),
    (256, 512, 64, False, 5),
    (257, 1056, 128, True, 8),        # a last group of 32
    (1000, 1184, 64, True, 9),        # half a group of 64 at the end
    (2000, 512, 32, False, 1),
    (2000, 2048, 256, False, 17),
    (513, 4096, 4096, True, 4),       # one group per row
    (5003, 1696, 128, True, 33),
    (20001, 2080, 32, True, 16),
    (33000, 4096, 128, False, 64),
    (300, 8192, 64, True, 70),        # more than one pass of batch rows
    (70000, 256, 128, True, 1),
])
@pytest.mark.parametrize("xt", DTYPES)
def test_shapes(pkg, eng, rows, cols, group, mins, nb, xt):
    import torch
    k = rows + cols + nb
    w = make(pkg, rows, cols, group, DTYPES[k % 3], mins, seed=k)
    x = torch.randn((nb, cols), generator=torch.Generator().manual_seed(k)).to(_dt(xt)).cuda()
    for yt in (xt, "f32"):
        check(w, x, eng.g4_matmul(w, x, out_dtype=_dt(yt)), f"{xt} -> {yt}")


@pytest.mark.gpu
@pytest.mark.parametrize("nb", list(range(1, 20)) + [31, 32, 47, 48, 49, 63, 64, 65, 128, 129])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_batch_size(pkg, eng, nb, group):
    import torch
    w = make(pkg, 401, 544, group, "bf16", nb % 2 == 1, seed=nb)
    x = torch.randn((nb, 544), generator=torch.Generator().manual_seed(nb)).cuda()
    check(w, x.bfloat16(), eng.g4_matmul(w, x.bfloat16()), "bf16")
    check(w, x, eng.g4_matmul(w, x), "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [200, 300, 333])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_many_batch_rows(pkg, eng, nb, group, xt):
    """More passes than the workspace is planned for one by one."""
    import torch
    w = make(pkg, 515, 288, group, "f16", True, seed=nb)
    x = torch.randn((nb, 288), generator=torch.Generator().manual_seed(nb)).to(_dt(xt)).cuda()
    fresh = pkg.Engine(0, max_rows=1, max_vocab=1024)
    try:
        check(w, x, fresh.g4_matmul(w, x, out_dtype=torch.float32))
    finally:
        fresh.close()


@pytest.mark.gpu
@pytest.mark.parametrize("st", DTYPES)
@pytest.mark.parametrize("xt", DTYPES)
@pytest.mark.parametrize("yt", DTYPES)
def test_types(pkg, eng, st, xt, yt):
    import torch
    w = make(pkg, 300, 384, 64, st, True, seed=5)
    x = torch.randn((6, 384), generator=torch.Generator().manual_seed(5)).to(_dt(xt)).cuda()
    check(w, x, eng.g4_matmul(w, x, out_dtype=_dt(yt)), f"{st} {xt} {yt}")


@pytest.mark.gpu
def test_fp32_activations_keep_their_low_bits(pkg, eng):
    """Activations that differ only below bfloat16's precision, and large and
    small ones side by side."""
    import torch
    w = make(pkg, 256, 256, 128, "f32", False, seed=2)
    x = 1.0 + torch.arange(256).float() * 2.0 ** -23
    check(w, x[None].cuda(), eng.g4_matmul(w, x[None].cuda()))
    x = torch.randn(256, generator=torch.Generator().manual_seed(1)) * 10.0 ** torch.linspace(-12, 12, 256)
    check(w, x[None].cuda(), eng.g4_matmul(w, x[None].cuda()))
    top = torch.full((256,), 3.0e37)                       # rounds up, not to infinity
    top[::2] = -3.0e37
    check(w, top[None].cuda(), eng.g4_matmul(w, top[None].cuda()))


@pytest.mark.gpu
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("nb", [1, 4, 12, 16])
def test_an_activation_much_larger_than_its_neighbours(pkg, eng, nb, mins):
    """Within the tolerance, and with few batch rows 2^-31 of the row's largest
    activation of 128 columns, times the magnitude of each weight of theirs."""
    import torch
    rows, cols, group = 700, 640, 64
    w = make(pkg, rows, cols, group, "f16", mins, seed=9)
    g = torch.Generator().manual_seed(9)
    x = torch.randn((nb, cols), generator=g)
    x[:, 5] = 3e6
    x[:, 300] = -2e8
    x = x.cuda()
    W, A = parts(w)
    xd = x.double()
    tol = (group + 3 * (cols // group) + 8) * 2.0 ** -23 * (xd.abs() @ A.t())
    if nb <= 12:
        top = xd.abs().reshape(nb, -1, 128).amax(2, keepdim=True).expand(nb, cols // 128, 128).reshape(nb, cols)
        tol = tol + 2.0 ** -31 * (top @ A.t())
    err = (eng.g4_matmul(w, x).double() - xd @ W.t()).abs()
    tol = tol + (xd @ W.t()).abs() * 2.0 ** -24
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.gpu
def test_strides_vectors_and_what_lies_behind(pkg, eng):
    import torch
    w = make(pkg, 333, 416, 128, "f16", True, seed=8)
    wide = torch.randn((5, 900), generator=torch.Generator().manual_seed(8)).half().cuda()
    for off in (0, 1, 7, 8):                               # rows that start anywhere
        x = wide[:, off:off + 416]
        buf = torch.full((5, 400), 7.0, device="cuda")
        y = buf[:, 3:336]
        assert eng.g4_matmul(w, x, out=y) is y
        check(w, x, y, f"offset {off}")
        assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 336:] == 7).all())
    t = torch.randn((416, 5), device="cuda").half().t()    # columns contiguous
    check(w, t, eng.g4_matmul(w, t))
    v = eng.g4_matmul(w, wide[0, :416])
    assert v.shape == (333,)
    check(w, wide[0, :416], v)
    assert eng.g4_matmul(w, wide[:0, :416]).shape == (0, 333)
    # rows of a vocabulary split: the same arrays from row 64 on
    part = pkg.G4Weights(w.q[64:], w.scales[:, 64:], w.mins[:, 64:], group=128)
    x = wide[:, :416]
    check(part, x, eng.g4_matmul(part, x))
    # weights whose rows are apart
    far = torch.zeros((333, 320), dtype=torch.uint8, device="cuda")
    far[:, :208] = w.q
    w2 = pkg.G4Weights(far[:, :208], w.scales, w.mins, group=128)
    assert torch.equal(eng.g4_matmul(w2, x), eng.g4_matmul(w, x))


@pytest.mark.gpu
def test_host_tensors(pkg, eng):
    import torch
    w = make(pkg, 777, 512, 64, "bf16", False, seed=4)
    for xt in DTYPES:
        x = torch.randn((3, 512), generator=torch.Generator().manual_seed(4)).to(_dt(xt))
        y = eng.g4_matmul(w, x)
        assert not y.is_cuda and torch.equal(y, eng.g4_matmul(w, x.cuda()).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,nb", [(20001, 2048, 3), (600, 8192, 16)])
def test_same_bits_and_batch_independence(pkg, eng, rows, cols, nb):
    import torch
    w = make(pkg, rows, cols, 128, "f16", True, seed=6)
    x = torch.randn((nb, cols), generator=torch.Generator().manual_seed(6)).cuda().half()
    y = eng.g4_matmul(w, x, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(y, eng.g4_matmul(w, x, out_dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("xt", DTYPES)
def test_non_finite_activations_stay_in_their_row(pkg, eng, xt):
    import torch
    w = make(pkg, 300, 512, 128, "f16", True, seed=9)
    x = torch.randn((4, 512), generator=torch.Generator().manual_seed(9)).to(_dt(xt)).cuda()
    bad = x.clone()
    bad[1, 100], bad[2, 511] = float("nan"), float("inf")
    y, z = eng.g4_matmul(w, x), eng.g4_matmul(w, bad)
    assert torch.equal(y[0], z[0]) and torch.equal(y[3], z[3])
    assert not bool(torch.isfinite(z[1:3]).any())


@pytest.mark.gpu
def test_streams_and_graphs(pkg, eng):
    import torch
    w = make(pkg, 3001, 1024, 128, "f16", False, seed=1)
    g = torch.Generator().manual_seed(1)
    x = torch.randn((2, 1024), generator=g).half().cuda()
    want = eng.g4_matmul(w, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = eng.g4_matmul(w, x)
    y2 = eng.g4_matmul(w, x.t().contiguous().t(), stream=side.cuda_stream)   # a copy is made on that stream
    side.synchronize()
    assert torch.equal(y, want) and torch.equal(y2, want)
    # a captured call, replayed on new inputs, also after a larger call has
    # made the workspace grow
    fresh = pkg.Engine(0, max_rows=8, max_vocab=4096)
    try:
        out = torch.empty_like(want)
        fresh.g4_matmul(w, x, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fresh.g4_matmul(w, x, out=out, check=False)
        big = torch.randn((64, 1024), generator=g).half().cuda()
        check(w, big, fresh.g4_matmul(w, big))
        for _ in range(3):
            x.copy_(torch.randn((2, 1024), generator=g).half())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eng.g4_matmul(w, x))
    finally:
        del graph
        fresh.close()


@pytest.mark.gpu
def test_device_refusals(pkg, eng):
    import torch
    lib = pkg.load()
    w = make(pkg, 64, 128, 32, "f16", True)
    x = torch.zeros((2, 128), device="cuda")
    y = torch.full((2, 64), 5.0, device="cuda")

    def call(struct=None, xt=0, ldx=128, nb=2, yt=0, ldy=64, flags=3, xp=None, yp=None):
        return lib.nls_g4_matmul(eng._h, ctypes.byref(struct or w.struct), xp or x.data_ptr(), xt, ldx, nb,
                                 yp or y.data_ptr(), yt, ldy, flags, None)

    def struct(**kw):
        s = pkg._abi.G4WeightsStruct.from_buffer_copy(w.struct)
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    for bad in (dict(xt=3), dict(yt=-1), dict(ldx=127), dict(ldy=63), dict(nb=-1), dict(flags=4), dict(flags=8),
                dict(xp=x.data_ptr() + 2), dict(yp=y.data_ptr() + 1)):
        assert call(**bad) == 1, bad
    for bad in (dict(q=None), dict(scales=None), dict(q=w.q.data_ptr() + 8), dict(scales=w.scales.data_ptr() + 2),
                dict(mins=w.mins.data_ptr() + 2), dict(rows=0), dict(cols=0), dict(cols=100), dict(group=16),
                dict(group=96), dict(group=192), dict(group=0), dict(stype=7), dict(q_ld=48), dict(q_ld=72),
                dict(s_ld=56), dict(s_ld=65)):
        assert call(struct(**bad)) == 1, bad
    assert call(nb=0) == 0
    torch.cuda.synchronize()
    assert bool((y == 5).all())
    with pytest.raises(ValueError):
        eng.g4_matmul(w, x[:, :96])
    with pytest.raises(ValueError):
        eng.g4_matmul(w, x, out=y[:, :32])
    with pytest.raises(ValueError):
        eng.g4_matmul(w, x, out=torch.empty((2, 64)))
    with pytest.raises(TypeError):
        eng.g4_matmul(w, x.double())


@pytest.mark.gpu
@pytest.mark.parametrize("big", [dict(cols=2**24 + 32), dict(cols=2**28), dict(cols=2**31 - 32), dict(rows=2**30 + 1),
                                 dict(rows=2**31 - 1)])
def test_sizes_past_the_range_are_refused(pkg, eng, big):
    import torch
    w = make(pkg, 64, 128, 32, "f16", True)
    s = pkg._abi.G4WeightsStruct.from_buffer_copy(w.struct)
    s.q_ld, s.s_ld = 2**31, 2**31
    for k, v in big.items():
        setattr(s, k, v)
    x = torch.zeros(128, device="cuda")
    assert pkg.load().nls_g4_matmul(eng._h, ctypes.byref(s), x.data_ptr(), 0, 2**31, 1, x.data_ptr(), 0, 2**31, 3, None) == 1


@pytest.mark.gpu
def test_the_default_stream_by_its_handle(pkg, eng):
    """stream=0 is the default stream, for temporaries and results too."""
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        with eng._on(True, 0):
            assert torch.cuda.current_stream() == torch.cuda.default_stream()
        with eng._on(True, side.cuda_stream):
            assert torch.cuda.current_stream().cuda_stream == side.cuda_stream
    w = make(pkg, 300, 256, 64, "f16", False)
    x = torch.randn((256, 3), device="cuda").t()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = eng.g4_matmul(w, x, stream=0)
    assert torch.equal(y, eng.g4_matmul(w, x))


@pytest.mark.gpu
def test_capture_that_would_have_to_allocate(pkg, eng):
    """Refused, and the capture goes on."""
    import torch
    w = make(pkg, 3001, 1024, 128, "f16", False, seed=1)
    x = torch.randn((2, 1024), device="cuda").half()
    out = torch.empty((2, 3001), dtype=torch.float16, device="cuda")
    other = pkg.Engine(0, max_rows=8, max_vocab=4096)
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            with pytest.raises(pkg.NlsError) as e:
                other.g4_matmul(w, x, out=out, check=False)
            out.zero_()
        assert e.value.status == pkg._abi.NLS_ERR_CAPACITY
        graph.replay()
        torch.cuda.synchronize()
        assert not bool(out.any())
        check(w, x, other.g4_matmul(w, x))
    finally:
        del graph
        other.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,nb", [(3001, 4096, 2), (40000, 512, 20)])
def test_a_wait_that_runs_out_is_an_error(pkg, eng, rows, cols, nb):
    import torch
    w = make(pkg, rows, cols, 128, "f16", True, seed=3)
    x = torch.randn((nb, cols), generator=torch.Generator().manual_seed(3)).half().cuda()
    want = eng.g4_matmul(w, x)
    for _ in range(2):
        eng.set_wait_limit(0)
        try:
            with pytest.raises(pkg.NlsError) as e:
                eng.g4_matmul(w, x)
        finally:
            eng.set_wait_limit(200 * 1000 * 1000)
        assert e.value.status == pkg._abi.NLS_ERR_TIMEOUT
        assert torch.equal(eng.g4_matmul(w, x), want)


@pytest.mark.gpu
@pytest.mark.parametrize("xt", DTYPES)
@pytest.mark.parametrize("group,mins", [(32, True), (64, False), (128, True)])
def test_bits_of_a_pass(pkg, eng, xt, group, mins):
    """Batch rows are taken in passes; a pass gives its rows the bits of a call
    of its own, and equal rows of a pass, wherever they stand in it, equal bits."""
    import torch
    per = 64 // max(1, 128 // group)
    if xt == "f32":
        per = min(per, 32)
    few = 4 if group == 32 or (group == 64 and xt != "f32") else 12
    w = make(pkg, 5003, 1184, group, "f16", mins, seed=7)
    g = torch.Generator().manual_seed(7)
    for nb in (few, few + 1, 9, per, per + few, per + few + 1, 2 * per + 3, 5 * per + 1):
        x = torch.randn((nb, 1184), generator=g).to(_dt(xt)).cuda()
        y = eng.g4_matmul(w, x, out_dtype=torch.float32)
        at = 0
        while at < nb:
            n = min(per, nb - at)
            if nb - at <= few:
                n = nb - at
            assert torch.equal(y[at:at + n], eng.g4_matmul(w, x[at:at + n], out_dtype=torch.float32)), (nb, at)
            turn = torch.arange(n).roll(n // 2 + 1)
            assert torch.equal(y[at:at + n][turn], eng.g4_matmul(w, x[at:at + n][turn], out_dtype=torch.float32))
            at += n


@pytest.mark.gpu
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("xt", DTYPES)
def test_groups_of_64_on_both_sides_of_their_ways(pkg, eng, xt, mins):
    """Groups of 64 leave the integer way after 4 batch rows of 16-bit
    activations and after 12 of fp32 ones."""
    import torch
    w = make(pkg, 2065, 1120, 64, "bf16", mins, seed=12)
    x = torch.randn((13, 1120), generator=torch.Generator().manual_seed(12)).to(_dt(xt)).cuda()
    y = [eng.g4_matmul(w, x[:nb], out_dtype=torch.float32) for nb in range(1, 14)]
    for nb in range(1, 14):
        check(w, x[:nb], y[nb - 1], f"{nb} rows")
    last = 12 if xt == "f32" else 4
    for nb in range(1, last):                              # one way: the same bits
        assert torch.equal(y[nb - 1][0], y[last - 1][0])
    assert not torch.equal(y[last - 1], y[last][:last])
