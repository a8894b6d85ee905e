"""iree_uk_amd_rmsnorm_pack and iree_uk_amd_gate_pack against their formulas in
64 bits. The reference has no such calls; what the tiles have to hold is the
reference's pack (tools/pack_test.c:13-58, no transposes) of the matrix that
the formula gives.

Tolerances count roundings of 2^-24 (f32) and one of the output's type. With u
and r as the kernels name them: a sum of squares of n columns is a sum of sums,
at most n / 64 + 16 terms one after the other, so r is off by half of that and
4 more; u has up to 2 roundings, u * r one, and the 8-bit forms 3 (the inverse,
the product, the scale). Activations: see `act_slack`."""
import math

import numpy as np
import pytest
import torch

from iree_amd import ukernel as uk

U32 = 2.0 ** -24
TYPES = {"f32": (torch.float32, uk.IN_TYPE_F32, uk.OUT_TYPE_F32), "f16": (torch.float16, uk.IN_TYPE_F16, uk.OUT_TYPE_F16),
         "bf16": (torch.bfloat16, uk.IN_TYPE_BF16, uk.OUT_TYPE_BF16)}
OUTS = {"s8": (torch.int8, uk.OUT_TYPE_S8), "f8": (torch.uint8, uk.OUT_TYPE_F8E4M3FN)}
ACTS = {"none": uk.ACTIVATION_NONE, "relu": uk.ACTIVATION_RELU, "gelu": uk.ACTIVATION_GELU,
        "gelu_tanh": uk.ACTIVATION_GELU_TANH, "silu": uk.ACTIVATION_SILU}
LARGEST = {"s8": 127.0, "f8": 448.0}
# eps / 2 of the type, and half of its smallest subnormal.
HALF = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}


def act64(x, act):
    if act == "relu":
        return np.where(x < 0, 0.0, x)
    if act == "silu":
        return x / (1 + np.exp(-x))
    if act == "gelu":
        return 0.5 * x * torch.special.erfc(torch.from_numpy(-x * math.sqrt(0.5))).numpy()
    if act == "gelu_tanh":  # (sigmoids: 1 + tanh loses the negative tail in 64 bits, too)
        return x / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x


def act_slack(x, act):
    """How far an activation may be off: 6 roundings, and one for each unit of the
    exponential's argument (t, or x^2 / 2 and its two roundings more); the
    approximation of erfc to 1.5e-7 beside, half of it times |x|. A sigmoid below 2^-126
    is the reciprocal of more than 2^126 and has no normal f32: the hardware's reciprocal
    gives zero for it, so |x| 2^-126 are lost at most (f32 GELU_TANH at x near -9: 1.8e-39 off, 9 * 2^-126 is 1.1e-37)."""
    y, a = np.abs(act64(x, act)), np.abs(x)
    if act == "silu":
        return y * (6 + 2 * a) * U32 + a * 2.0 ** -126
    if act == "gelu_tanh":
        return y * (6 + 4 * (1.6 * a + 0.0714 * a ** 3)) * U32 + a * 2.0 ** -126
    if act == "gelu":
        return y * (8 + 3 * a * a) * U32 + a * (0.75e-7 + 6 * U32)
    return 0 * a


def f8_value(bits):
    return torch.as_tensor(bits).view(torch.float8_e4m3fn).to(torch.float64).numpy()


def tiles_to_matrix(t):
    M1, K1, M0, K0 = t.shape
    return t.transpose(0, 2, 1, 3).reshape(M1 * M0, K1 * K0)


class Call:
    """Buffers of a call inside larger ones whose other bytes have to stay."""

    def __init__(self, seed):
        self.rng = np.random.default_rng(seed)

    def matrix(self, rows, cols, dtype, pitch, offset, values=None, device="cuda"):
        full = torch.full((offset + rows * pitch + 7,), 3.0, dtype=torch.float32)
        if values is not None:
            v = torch.from_numpy(np.ascontiguousarray(values)).to(torch.float32)
            full[offset:offset + rows * pitch].view(rows, pitch)[:, :cols] = v
        return full.to(dtype).to(device)

    def values(self, rows, cols):
        return self.rng.standard_normal((rows, cols)) * np.exp(0.7 * self.rng.standard_normal(cols))


def same_bytes(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


def view(t, rows, cols, pitch, offset):
    return t[offset:offset + rows * pitch].view(rows, pitch)[:, :cols] if rows else t[:0].view(0, cols)


def check_rows(y, y_slack, tin, tout, tiles, scale, rows, cols, name):
    """The tiles (and scales) against the formula's y in 64 bits, known to y_slack."""
    got = tiles_to_matrix(tiles)
    assert not got[rows:].any() and not got[:, cols:].any(), name   # zeros where tiles reach beyond
    got = got[:rows, :cols]
    if tout not in LARGEST:
        half, tiny = HALF[tin]
        off = np.abs(got - y) - (np.abs(y) * half + tiny + y_slack * (1 + half))
        assert off.max(initial=-1) <= 0, (name, off.max())
        return
    largest = LARGEST[tout]
    top = np.abs(y).max(axis=1, initial=0.0)
    # The largest |y| is off by at most the most that any y of its row is.
    rel = np.where(top > 0, (y_slack.max(axis=1, initial=0.0)) / np.where(top > 0, top, 1), 0) + 3 * U32
    assert np.all(np.abs(scale - top / largest) <= top / largest * rel), name
    v = y / np.where(top > 0, top / largest, 1)[:, None]
    slack = (y_slack / np.where(top > 0, top / largest, 1)[:, None]) + np.abs(v) * (rel[:, None] + 3 * U32)
    if tout == "s8":
        half = 0.5
    else:
        half = np.exp2(np.floor(np.log2(np.maximum(np.abs(v) + slack, 2.0 ** -6))) - 4)
    off = np.abs(got - v) - (half + slack)
    assert off.max(initial=-1) <= 0, (name, off.max())


def norm_reference(x, res, w, eps, cols):
    h = x + res if res is not None else x
    u = h * w if w is not None else h
    y = u / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps)
    # h: one rounding of what is added (its own and, behind a cancellation, none more: both
    # addends are exact), r: half the sum's, and the rest.
    c = 2 + (cols / 64 + 16) / 2 + 4 + 1
    return h, y, np.abs(y) * c * U32


def run_norm(lib, tin, tout, rows, cols, M0, K0, *, residual, with_sum, weight, in_place=None, pitch=0, offset=0, M1=None,
             K1=None, eps=1e-5, device="cuda", values=None, seed=0):
    c = Call(seed)
    dt, fin, fout = TYPES[tin]
    ot, fo = OUTS.get(tout, (dt, fout))
    M1 = -(-rows // M0) if M1 is None else M1
    K1 = -(-cols // K0) if K1 is None else K1
    pin, pres, psum = cols + pitch, cols + 2 * pitch, cols + 3 * pitch
    x = c.matrix(rows, cols, dt, pin, offset, c.values(rows, cols) if values is None else values, device)
    res = c.matrix(rows, cols, dt, pres, offset + 1, 2 * c.values(rows, cols), device) if residual else None
    w = torch.from_numpy(1 + 0.2 * c.rng.standard_normal(cols)).to(torch.float32).to(dt).to(device) if weight else None
    x0, r0 = x.cpu().clone(), res.cpu().clone() if residual else None
    if in_place == "in":
        total, psum, so = x, pin, offset
    elif in_place == "residual":
        total, psum, so = res, pres, offset + 1
    else:
        total, so = (c.matrix(rows, cols, dt, psum, offset + 2, None, device) if with_sum else None), offset + 2
    t0 = total.cpu().clone() if total is not None else None
    n = M1 * K1 * M0 * K0
    stride = K1 * M0 * K0 + 3 * pitch
    out = torch.full((offset + M1 * stride + 5,), 5, dtype=ot, device=device)
    scale = torch.full((rows + 2,), -7.0, device=device)
    lib.rmsnorm_pack(x.data_ptr(), offset, pin, res.data_ptr() if residual else None, offset + 1, pres,
                     total.data_ptr() if total is not None else None, so, psum, w.data_ptr() if weight else None, eps,
                     out.data_ptr(), offset, stride, scale.data_ptr() if tout in LARGEST else None, rows, cols, M1, K1, M0,
                     K0, fin | fo)
    lib.synchronize()
    xv = view(x0, rows, cols, pin, offset).double().numpy()
    rv = view(r0, rows, cols, pres, offset + 1).double().numpy() if residual else None
    wv = w.cpu().double().numpy() if weight else None
    name = (tin, tout, rows, cols, M0, K0, residual, weight, in_place, pitch, offset)
    h, y, slack = norm_reference(xv, rv, wv, eps, max(cols, 1))
    out = out.cpu()
    raw = torch.stack([out[offset + i * stride:offset + i * stride + K1 * M0 * K0] for i in range(M1)]) if M1 else out[:0]
    vals = f8_value(raw) if tout == "f8" else raw.double().numpy()
    # What the call has no business with is as it was.
    mask = torch.ones(out.numel(), dtype=torch.bool)
    for i in range(M1):
        mask[offset + i * stride:offset + i * stride + K1 * M0 * K0] = False
    assert bool((out[mask] == 5).all()), name
    sc = scale.cpu().double().numpy()
    assert np.all(sc[rows if tout in LARGEST else 0:] == -7.0), name
    if total is not None:
        t1 = total.cpu()
        got = view(t1, rows, cols, psum, so).double().numpy()
        half, tiny = HALF[tin]
        assert np.all(np.abs(got - h) <= np.abs(h) * (half + U32) * (1 + half) + tiny), name
        t1v = t1.clone()
        view(t1v, rows, cols, psum, so).copy_(view(t0, rows, cols, psum, so))
        assert same_bytes(t1v, t0), name
    if total is not x:
        assert same_bytes(x, x0)
    if residual and total is not res:
        assert same_bytes(res, r0)
    assert n == vals.size
    return y, slack, vals.reshape(M1, K1, M0, K0), sc[:rows], name


SIZES = [  # rows, cols, M0, K0
    (1, 1, 1, 16), (1, 64, 1, 16), (3, 17, 16, 16), (5, 100, 32, 8), (33, 127, 16, 32), (16, 1024, 16, 16),
    (7, 1021, 4, 3), (2, 4096, 1, 32), (9, 2050, 8, 1), (18, 5001, 16, 8), (2, 16385, 16, 16), (1, 41003, 16, 4),
    (1, 131077, 1, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("tin", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tout", ["s8", "f8", "same"])
def test_norm_of_many_sizes(gpu, tin, tout):
    lib, _ = gpu
    tout = tin if tout == "same" else tout
    for i, (rows, cols, M0, K0) in enumerate(SIZES):
        y, slack, tiles, scale, name = run_norm(lib, tin, tout, rows, cols, M0, K0, residual=i % 3 != 0, with_sum=i % 3 == 1,
                                                weight=i % 4 != 3, pitch=(0, 1, 8)[i % 3], offset=(0, 3)[i % 2], seed=i)
        check_rows(y, slack, tin, tout, tiles, scale, rows, cols, name)


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", ["in", "residual"])
@pytest.mark.parametrize("rows,cols", [(1, 333), (40, 4096), (2, 20000), (1, 70001)])
def test_norm_writes_the_sum_over_one_of_its_inputs(gpu, in_place, rows, cols):
    lib, _ = gpu
    for tin in ("bf16", "f32"):
        y, slack, tiles, scale, name = run_norm(lib, tin, "s8", rows, cols, 16, 16, residual=True, with_sum=True, weight=True,
                                                in_place=in_place, pitch=4, offset=1, seed=5)
        check_rows(y, slack, tin, "s8", tiles, scale, rows, cols, name)


@pytest.mark.gpu
def test_norm_fills_tiles_beyond_the_matrix_with_zeros(gpu):
    """More tiles than the matrix needs, in both directions, and matrices without rows or columns."""
    lib, _ = gpu
    for tout in ("s8", "f8", "bf16"):
        for rows, cols, M1, K1 in [(5, 70, 3, 9), (0, 70, 2, 5), (16, 16, 2, 300), (0, 0, 0, 3)]:
            y, slack, tiles, scale, name = run_norm(lib, "bf16", tout, rows, cols, 16, 16, residual=False, with_sum=False,
                                                    weight=True, M1=M1, K1=K1)
            check_rows(y, slack, "bf16", tout, tiles, scale, rows, cols, name)
    tiles = torch.full((2, 3, 16, 16), 9, dtype=torch.int8, device="cuda")
    scale = torch.full((20,), 9.0, device="cuda")
    one = torch.zeros(16, device="cuda")
    lib.rmsnorm_pack(one.data_ptr(), 0, 0, None, 0, 0, None, 0, 0, None, 1e-5, tiles.data_ptr(), 0, 768, scale.data_ptr(), 20,
                     0, 2, 3, 16, 16, uk.IN_TYPE_F32 | uk.OUT_TYPE_S8)   # 20 rows of no columns
    lib.synchronize()
    assert not tiles.any() and not scale.any()


def special_rows(cols):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((8, cols))
    x[1] = 0
    x[2, cols // 2] = np.nan
    x[3, cols - 1] = np.inf
    x[4, 0] = -np.inf
    x[5] = 1e-36
    x[6] = 0
    x[6, cols // 3] = 2.0 ** -126
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("tout", ["s8", "f8"])
@pytest.mark.parametrize("cols", [65, 4096, 50000])
def test_rows_without_an_8_bit_form(gpu, tout, cols):
    """Zeros and next to nothing: scale 0. NaN and infinities: scale NaN. The row is zeros either way,
    and its neighbours are what they are without it."""
    lib, _ = gpu
    for tin in ("bf16", "f32"):
        x = special_rows(cols)
        y, slack, tiles, scale, name = run_norm(lib, tin, tout, 8, cols, 16, 16, residual=False, with_sum=False, weight=False,
                                                values=x)
        rows = tiles_to_matrix(tiles)[:8, :cols]
        assert np.isnan(scale[2:5]).all() and not rows[2:5].any()
        assert not scale[[1, 5, 6]].any() and not rows[[1, 5, 6]].any(), scale
        keep = [0, 7]
        check_rows(y[keep], slack[keep], tin, tout, tiles[:, :, keep, :], scale[keep], 2, cols, name)
        dt, fin, _ = TYPES[tin]
        g = torch.from_numpy(x).to(torch.float32).to(dt).cuda()
        out = torch.empty(1, -(-cols // 16), 16, 16, dtype=torch.int8, device="cuda")
        sc = torch.empty(8, device="cuda")
        lib.gate_pack(g.data_ptr(), 0, cols, None, 0, 0, out.data_ptr(), 0, out.stride(0), sc.data_ptr(), 8, cols,
                      *out.shape, fin | OUTS[tout][1])
        lib.synchronize()
        sc = sc.cpu().numpy()
        rows = tiles_to_matrix(out.cpu().numpy())[:8]
        assert np.isnan(sc[2:5]).all() and not sc[[1, 5, 6]].any() and not rows[1:7].any()
        assert rows[0].any() and rows[7].any()


@pytest.mark.gpu
def test_norm_of_a_row_that_no_sum_of_squares_holds(gpu):
    """1e30 squared is beyond f32: NaN scales, and NaN where the output is not quantized."""
    lib, _ = gpu
    x = torch.full((2, 96), 1e30, device="cuda")
    x[1] = 1.0
    s = torch.empty(2, device="cuda")
    q = torch.empty(1, 6, 16, 16, dtype=torch.int8, device="cuda")
    lib.rmsnorm_pack(x.data_ptr(), 0, 96, None, 0, 0, None, 0, 0, None, 0.0, q.data_ptr(), 0, 0, s.data_ptr(), 2, 96, 1, 6, 16,
                     16, uk.IN_TYPE_F32 | uk.OUT_TYPE_S8)
    y = torch.empty(2, 96, device="cuda")
    lib.rmsnorm_pack(x.data_ptr(), 0, 96, None, 0, 0, None, 0, 0, None, 0.0, y.data_ptr(), 0, 96, None, 2, 96, 2, 6, 1, 16,
                     uk.IN_TYPE_F32 | uk.OUT_TYPE_F32)
    lib.synchronize()
    assert math.isnan(s[0].item()) and not q[0, :, 0].any() and bool((q[0, :, 1] == 127).all())
    assert bool(y[0].isnan().all()) and torch.allclose(y[1], torch.ones_like(y[1]), rtol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("tin", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tout", ["s8", "f8", "same"])
@pytest.mark.parametrize("act", list(ACTS))
def test_gate_of_many_sizes(gpu, tin, tout, act):
    lib, _ = gpu
    tout = tin if tout == "same" else tout
    dt, fin, fout = TYPES[tin]
    ot, fo = OUTS.get(tout, (dt, fout))
    for i, (rows, cols, M0, K0) in enumerate(SIZES):
        c = Call(100 + i)
        up = i % 3 != 2
        offset, pitch = (0, 3)[i % 2], (2 if up else 1) * cols + (0, 5)[i % 2]
        both = np.concatenate([c.values(rows, cols), c.values(rows, cols)], axis=1)[:, :(2 if up else 1) * cols]
        if act == "none":
            both[0, 0] = -both[0, 0]
        m = c.matrix(rows, both.shape[1], dt, pitch, offset, both)
        M1, K1 = -(-rows // M0), -(-cols // K0)
        out = torch.full((M1, K1, M0, K0), 5, dtype=ot, device="cuda")
        scale = torch.full((rows + 1,), -7.0, device="cuda")
        lib.gate_pack(m.data_ptr(), offset, pitch, m.data_ptr() if up else None, offset + cols, pitch, out.data_ptr(), 0,
                      out.stride(0), scale.data_ptr() if tout in LARGEST else None, rows, cols, M1, K1, M0, K0,
                      fin | fo | ACTS[act])
        lib.synchronize()
        halves = view(m, rows, both.shape[1], pitch, offset).cpu().double().numpy()
        g, u = halves[:, :cols], halves[:, cols:] if up else 1.0
        y = act64(g, act) * u
        slack = act_slack(g, act) * np.abs(u) + np.abs(y) * U32
        name = (tin, tout, act, rows, cols, M0, K0)
        t = out.cpu()
        check_rows(y, slack, tin, tout, f8_value(t) if tout == "f8" else t.double().numpy(),
                   scale.cpu().double().numpy()[:rows], rows, cols, name)
        assert scale[rows].item() == -7.0


@pytest.mark.gpu
def test_row_ops_on_host_memory(gpu):
    """Ordinary memory is staged, as for every entry point; in place, too."""
    lib, _ = gpu
    for in_place in (None, "in", "residual"):
        y, slack, tiles, scale, name = run_norm(lib, "bf16", "f8", 21, 300, 16, 32, residual=True, with_sum=True, weight=True,
                                                in_place=in_place, pitch=3, offset=2, device="cpu")
        check_rows(y, slack, "bf16", "f8", tiles, scale, 21, 300, name)
    g = torch.randn(5, 40)
    out = torch.zeros(5, 40)
    lib.gate_pack(g.data_ptr(), 0, 40, None, 0, 0, out.data_ptr(), 0, 40, None, 5, 40, 5, 10, 1, 4,
                  uk.IN_TYPE_F32 | uk.OUT_TYPE_F32)
    assert torch.equal(out, g)


@pytest.mark.gpu
def test_row_ops_in_a_captured_graph_and_on_a_side_stream(gpu):
    lib, _ = gpu
    x = torch.randn(40, 1000, device="cuda").to(torch.bfloat16)
    s = torch.cuda.Stream()
    outs = [torch.empty(3, 63, 16, 16, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty(40, device="cuda") for _ in range(2)]

    def call(i):
        lib.rmsnorm_pack(x.data_ptr(), 0, 1000, None, 0, 0, None, 0, 0, None, 1e-5, outs[i].data_ptr(), 0, outs[i].stride(0),
                         scales[i].data_ptr(), 40, 1000, 3, 63, 16, 16, uk.IN_TYPE_BF16 | uk.OUT_TYPE_S8)

    try:
        lib.set_pointer_mode(uk.POINTER_MODE_DEVICE)
        torch.cuda.synchronize()
        lib.set_stream(s.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(0)
        for k in range(3):
            x.copy_(torch.randn(40, 1000, device="cuda") * (k + 1))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            call(1)
            s.synchronize()
            assert torch.equal(*outs) and torch.equal(*scales)
    finally:
        lib.set_stream(None)
        lib.set_pointer_mode(uk.POINTER_MODE_AUTO)


def test_row_op_refusals(lib):
    """Needs no device: what the header rules out is a contract violation."""
    lib.raise_on_violation(True)

    def norm(flags=uk.IN_TYPE_BF16 | uk.OUT_TYPE_S8, rows=16, cols=32, M1=1, K1=2, M0=16, K0=16, scale=64, residual=None,
             total=None, stride=32, eps=1e-5, src=64, dst=64, total_stride=32, out_stride=512):
        lib.rmsnorm_pack(src, 0, stride, residual, 0, 32, total, 0, total_stride, None, eps, dst, 0, out_stride, scale, rows,
                         cols, M1, K1, M0, K0, flags)

    bad = [dict(flags=uk.IN_TYPE_BF16), dict(flags=uk.OUT_TYPE_S8), dict(flags=uk.IN_TYPE_BF16 | uk.OUT_TYPE_F16),
           dict(flags=uk.IN_TYPE_F32 | uk.OUT_TYPE_BF16), dict(flags=0x02 | uk.OUT_TYPE_S8),
           dict(flags=uk.IN_TYPE_BF16 | uk.OUT_TYPE_S8 | uk.ACTIVATION_SILU), dict(flags=0x10000 | 0x25),
           dict(rows=17), dict(cols=33), dict(rows=-1), dict(M1=-1), dict(K0=1 << 15), dict(M1=1 << 31),
           dict(M1=1 << 30, M0=16), dict(scale=None), dict(total=64), dict(stride=-32), dict(eps=-1.0),
           dict(eps=float("nan")), dict(M0=64, K0=128, K1=1), dict(src=None), dict(dst=None), dict(M1=2, out_stride=511),
           dict(residual=64, total=64, total_stride=31)]
    for kw in bad:
        with pytest.raises(uk.ContractViolation):
            norm(**kw)
    norm(rows=0, M1=0)

    def gate(flags):
        lib.gate_pack(64, 0, 32, None, 0, 0, 64, 0, 512, 64, 16, 32, 1, 2, 16, 16, flags)

    for flags in (uk.IN_TYPE_BF16 | uk.OUT_TYPE_S8 | 0x500, uk.IN_TYPE_F16 | uk.OUT_TYPE_F32, 0):
        with pytest.raises(uk.ContractViolation):
            gate(flags)


@pytest.mark.gpu
@pytest.mark.parametrize("m0,k0,cols", [(16, 16, 13), (1, 8, 8), (24, 4, 20)])
def test_more_rows_than_a_launch_takes(lib, m0, k0, cols):
    """2^21 rows of tiles are a launch: a call of more gives what calls of fewer give, byte by byte."""
    lib.raise_on_violation(True)
    rows = (1 << 21) + 1003
    M1, K1 = -(-rows // m0), -(-cols // k0)
    panel = K1 * m0 * k0
    g = torch.Generator(device="cuda").manual_seed(rows + m0)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(torch.bfloat16)
    y = torch.randn(rows, cols, generator=g, device="cuda").to(torch.bfloat16)
    flags = uk.IN_TYPE_BF16 | uk.OUT_TYPE_S8
    px, py = x.data_ptr(), y.data_ptr()

    def run(part, norm):
        tiles = torch.full((M1 * panel,), 7, dtype=torch.int8, device="cuda")
        total = torch.full((rows, cols), 3.0, dtype=torch.bfloat16, device="cuda")
        scale = torch.full((rows,), 5.0, device="cuda")
        for m in range(0, M1, part):
            first, panels = m * m0, min(part, M1 - m)
            here = min(rows - first, panels * m0)
            if norm:
                lib.rmsnorm_pack(px, first * cols, cols, py, first * cols, cols, total.data_ptr(), first * cols, cols, None,
                                 1e-5, tiles.data_ptr(), m * panel, panel, scale[first:].data_ptr(), here, cols, panels, K1,
                                 m0, k0, flags)
            else:
                lib.gate_pack(px, first * cols, cols, py, first * cols, cols, tiles.data_ptr(), m * panel, panel,
                              scale[first:].data_ptr(), here, cols, panels, K1, m0, k0, flags | uk.ACTIVATION_SILU)
        torch.cuda.synchronize()
        return tiles, total, scale

    for norm in (True, False):
        for a, b in zip(run(M1, norm), run(100000 // m0, norm)):
            assert same_bytes(a, b), norm


@pytest.mark.gpu
@pytest.mark.parametrize("tin", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cols", [100, 70001])
def test_gates_of_the_lowest_numbers_are_zero(gpu, tin, cols):
    """What a mask puts into a gate: every activation makes zeros of it, and the row's scale is that of its other columns.
    -infinity: zero, or NaN where the formula multiplies it by zero."""
    lib, _ = gpu
    dt, fin, fout = TYPES[tin]
    low = torch.finfo(dt).min
    g = torch.Generator().manual_seed(3)
    gate = torch.randn(4, cols, generator=g).to(dt)
    gate[0, 1::3] = low
    gate[1, :] = low
    gate[2, 5] = low / 4
    gate[2, 7] = -60000.0
    gate[3, 2] = -float("inf")
    masked = [gate[0] == low, gate[1] == low, gate[2] < -1000]
    up = torch.randn(4, cols, generator=g).to(dt).cuda()
    K1 = -(-cols // 16)
    x = gate.cuda()
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        kept = act64(gate.double().numpy()[:3], act) * up[:3].cpu().double().numpy()
        top = np.abs(np.where(torch.stack(masked).numpy(), 0.0, kept)).max(axis=1)
        for tout, fo in ((tin, fout), ("s8", uk.OUT_TYPE_S8)):
            tiles = torch.zeros(K1 * 16 * 4, dtype=torch.int8 if tout == "s8" else dt, device="cuda")
            scale = torch.zeros(4, device="cuda")
            lib.gate_pack(x.data_ptr(), 0, cols, up.data_ptr(), 0, cols, tiles.data_ptr(), 0, K1 * 16, scale.data_ptr(), 4, cols,
                          4, K1, 1, 16, fin | fo | ACTS[act])
            lib.synchronize()
            got = tiles.cpu().double().view(4, K1 * 16)[:, :cols]
            for row, m in enumerate(masked):
                assert not got[row][m].any(), (act, tout, row)
            assert got[0][~masked[0]].any() and got[2].any() and not got[:3].isnan().any(), (act, tout)
            limit = act in ("relu", "gelu")
            if tout == "s8":
                # (1e-5: the activation's own 2e-6 at most, and the scale's roundings)
                assert np.allclose(scale[:3].cpu().numpy(), top / 127, rtol=1e-5, atol=0), (act, scale, top / 127)
                assert scale[3].isnan().item() != limit and got[3].any().item() == limit
            else:
                assert got[3, 2].isnan().item() != limit and (not limit or got[3, 2] == 0)


@pytest.mark.gpu
def test_epilogues_of_the_lowest_numbers_are_zero(gpu):
    """A bias of the lowest number masks a column: zeros, with every activation, beside a residual, too."""
    lib, _ = gpu
    a = torch.ones(2, 4, 16, 16, dtype=torch.int8, device="cuda")
    b = torch.ones(3, 4, 16, 16, dtype=torch.int8, device="cuda")
    bias = torch.zeros(48, device="cuda")
    bias[7] = torch.finfo(torch.float32).min
    bias[40] = -1e30
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        for mode in (uk.KERNEL_MODE_AUTO, uk.KERNEL_MODE_GENERIC):
            lib.set_kernel_mode(mode)
            try:
                out = torch.full((32, 48), 2.0, device="cuda")
                lib.mmt4d_epilogue_unpack(a.data_ptr(), 0, a.stride(0), b.data_ptr(), 0, b.stride(0), out.data_ptr(), 0, 48,
                                          out.data_ptr(), 0, 48, 32, 48, None, None, bias.data_ptr(), 2, 3, 4, 16, 16, 16,
                                          uk.MMT4D_TYPE_S8S8S32, uk.OUT_TYPE_F32 | ACTS[act])
                lib.synchronize()
            finally:
                lib.set_kernel_mode(uk.KERNEL_MODE_AUTO)
            other = torch.ones(48, dtype=torch.bool)
            other[7] = other[40] = False
            assert bool((out[:, 7] == 2).all()) and bool((out[:, 40] == 2).all()) and bool((out.cpu()[:, other] == 66).all()), act


@pytest.mark.gpu
@pytest.mark.parametrize("tin", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cols", [5, 65, 4093, 32769])
def test_norm_padding_is_zero_whatever_the_rows_hold(gpu, tin, cols):
    """Into the in type: rows of tiles beyond the matrix and columns beyond a row are zeros also where nothing is added to
    the mean of squares, and beside rows that have no norm; those are NaN themselves. Rows in registers and longer ones."""
    lib, _ = gpu
    x = np.random.default_rng(cols).standard_normal((6, cols))
    x[1] = 0
    x[2, cols // 2] = np.nan
    x[3, cols - 1] = -np.inf
    x[4] = 1e30   # (f16: infinity)
    for eps in (0.0, 1e-5):
        y, slack, tiles, _, name = run_norm(lib, tin, tin, 6, cols, 8, 16, residual=False, with_sum=False, weight=True,
                                            values=x, M1=2, K1=-(-cols // 16) + 2, eps=eps)
        got = tiles_to_matrix(tiles)
        assert not got[6:].any() and not got[:, cols:].any(), name
        assert np.isnan(got[2:5, :cols]).all(), name
        assert np.isnan(got[1, :cols]).all() if eps == 0 else not got[1].any(), name
        keep = [0, 5]
        check_rows(y[keep], slack[keep], tin, tin, tiles[:1][:, :, keep, :], None, 2, cols, name)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [70, 40000])
def test_norm_forms_the_weighted_row_before_it_divides(gpu, cols):
    """Weights that take h beyond f32, or below what has an inverse: infinities and scales of NaN and 0, as the header says,
    where the quotient times the weight would be a number. Squares that f32 does not hold: NaN."""
    lib, _ = gpu
    K1 = -(-cols // 16)
    for h, w, value, scale in [(1e15, 1e30, math.inf, math.nan), (2.0 ** -60, 2.0 ** -55, 2.0 ** -55, 0.0), (1e20, 1.0, math.nan, math.nan),
                               (2.0 ** -60, 2.0 ** -45, 2.0 ** -45, 2.0 ** -45 / 127)]:
        x = torch.full((2, cols), h, device="cuda")
        weight = torch.full((cols,), w, device="cuda")
        y = torch.full((2, K1, 1, 16), 7.0, device="cuda")
        q = torch.full((2, K1, 1, 16), 7, dtype=torch.int8, device="cuda")
        s = torch.full((2,), 7.0, device="cuda")
        for out, fo in ((y, uk.OUT_TYPE_F32), (q, uk.OUT_TYPE_S8)):
            lib.rmsnorm_pack(x.data_ptr(), 0, cols, None, 0, 0, None, 0, 0, weight.data_ptr(), 0.0, out.data_ptr(), 0,
                             out.stride(0), s.data_ptr(), 2, cols, 2, K1, 1, 16, uk.IN_TYPE_F32 | fo)
        lib.synchronize()
        # (the sum of squares is off by cols / 64 roundings and the scale by a few)
        same = dict(rtol=(cols / 64 + 32) * U32, atol=0.0, equal_nan=True)
        assert np.allclose(y.cpu().numpy().reshape(2, -1)[:, :cols], value, **same), (h, w)
        assert np.allclose(s.cpu().numpy(), scale, **same), (h, w, s)
        assert bool((q.view(2, -1)[:, :cols] == (127 if scale > 0 else 0)).all()) and not q.view(2, -1)[:, cols:].any(), (h, w)
        assert not y.view(2, -1)[:, cols:].any(), (h, w)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [200, 40000])
@pytest.mark.parametrize("on", ["cuda", "cpu"])
def test_inputs_of_one_row_for_all(gpu, cols, on):
    """A stride of 0: the same row of x beside every row of the residual, the same gate beside every row of up."""
    lib, _ = gpu
    g = torch.Generator().manual_seed(cols)
    one, many = torch.randn(1, cols, generator=g).to(on), torch.randn(5, cols, generator=g).to(on)
    all_ = one.expand(5, cols).contiguous()
    K1 = -(-cols // 16)

    def run(first, second, strides, norm):
        q = torch.full((1, K1, 16, 16), 7, dtype=torch.int8, device=on)
        s, total = torch.full((5,), 7.0, device=on), torch.full((5, cols), 7.0, device=on)
        args = (first.data_ptr(), 0, strides[0], second.data_ptr(), 0, strides[1])
        into = (q.data_ptr(), 0, q.numel(), s.data_ptr(), 5, cols, 1, K1, 16, 16, uk.IN_TYPE_F32 | uk.OUT_TYPE_S8)
        if norm:
            lib.rmsnorm_pack(*args, total.data_ptr(), 0, cols, None, 1e-5, *into)
        else:
            lib.gate_pack(*args, *into[:-1], into[-1] | uk.ACTIVATION_SILU)
        lib.synchronize()
        return q, s, total

    for norm in (True, False):
        for wide, narrow in ((run(all_, many, (cols, cols), norm), run(one, many, (0, cols), norm)),
                             (run(many, all_, (cols, cols), norm), run(many, one, (cols, 0), norm))):
            assert all(torch.equal(a, b) for a, b in zip(wide, narrow)), (norm, cols, on)
            assert wide[0].any() and (wide[1] > 0).all()
