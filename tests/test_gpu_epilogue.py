"""iree_uk_amd_mmt4d_epilogue_unpack against its formula in 64 bits: the product
(mmt4d.c:55-114 without an accumulator input), scales, bias, activation and
residual. The reference has no such call.

Operands are small integers, so that the products' sums are exact in 32 bits
whatever their order; what is left are the roundings of 2^-24 of the
conversion, of each factor, of the sums and of the activation, and one of the
output's type."""
import numpy as np
import pytest
import torch

from iree_amd import ukernel as uk
from test_gpu_row_ops import ACTS, HALF, U32, act64, act_slack

# mmt4d type -> (operand kinds, bytes of what holds them)
S8, F8, F16, BF16, F32 = (uk.MMT4D_TYPE_S8S8S32, uk.MMT4D_TYPE_F8E4M3FNF8E4M3FNF32, uk.MMT4D_TYPE_F16F16F32,
                          uk.MMT4D_TYPE_BF16BF16F32, uk.MMT4D_TYPE_F32F32F32)
TORCH = {S8: torch.int8, F8: torch.float8_e4m3fn, F16: torch.float16, BF16: torch.bfloat16, F32: torch.float32,
         uk.MMT4D_TYPE_S16S16S32: torch.int16}
OUTS = {"f32": (torch.float32, uk.OUT_TYPE_F32), "f16": (torch.float16, uk.OUT_TYPE_F16),
        "bf16": (torch.bfloat16, uk.OUT_TYPE_BF16)}


def tiled(x, t0, k0, t1, k1, dtype):
    """A rows x k matrix of integers in tiles; what the tiles hold beyond it must not matter to it, so not zeros
    beyond the rows; zeros beyond k."""
    full = torch.full((t1 * t0, k1 * k0), 1.0)
    full[:, x.shape[1]:] = 0
    full[:x.shape[0], :x.shape[1]] = torch.from_numpy(x).float()
    t = full.view(t1, t0, k1, k0).transpose(1, 2).contiguous()
    return t.to(dtype).cuda()


def run(lib, type_, rows, cols, k, M0, N0, K0, out, act, *, scales=True, bias=True, residual=None, pitch=0, offset=0,
        flags=0, seed=0, capture=None):
    """One call between guards, and its distance from the formula. `residual`: None, "own" or "in place"."""
    rng = np.random.default_rng(seed)
    M1, N1, K1 = -(-rows // M0), -(-cols // N0), -(-k // K0)
    a = rng.integers(-4, 5, (rows, k)).astype(np.float64)
    b = rng.integers(-4, 5, (cols, k)).astype(np.float64)
    lhs, rhs = tiled(a, M0, K0, M1, K1, TORCH[type_]), tiled(b, N0, K0, N1, K1, TORCH[type_])
    dt, fo = OUTS[out]
    width = 10 / (6.0 * np.sqrt(max(k, 1)))
    rs = torch.from_numpy((0.2 + rng.random(rows)) * 0.4).float().cuda() if scales else None
    cs = torch.from_numpy((0.2 + rng.random(cols)) * width).float().cuda() if scales else None
    bi = torch.from_numpy(rng.standard_normal(cols)).float().cuda() if bias else None
    op, rp = cols + pitch, cols + 2 * pitch
    buf = torch.from_numpy(rng.standard_normal(offset + rows * op + 9)).to(dt).cuda()
    res = torch.from_numpy(2 * rng.standard_normal(offset + 2 + rows * rp)).to(dt).cuda()
    before = buf.cpu().clone()
    res_at, res_off = (buf, offset) if residual == "in place" else (res, offset + 1)
    rp = op if residual == "in place" else rp

    def at(t, pitch_, off):
        return t[off:off + rows * pitch_].view(rows, pitch_)[:, :cols]

    r64 = at(res_at, rp, res_off).cpu().double().numpy().copy() if residual else 0.0

    def call():
        lib.mmt4d_epilogue_unpack(
            lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(),
            res_at.data_ptr() if residual else None, res_off, rp, buf.data_ptr(), offset, op, rows, cols,
            rs.data_ptr() if scales else None, cs.data_ptr() if scales else None, bi.data_ptr() if bias else None, M1, N1, K1,
            M0, N0, K0, type_ | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION | flags, fo | ACTS[act])
    if capture:
        capture(call)
    else:
        call()
        lib.synchronize()
    name = (type_, rows, cols, k, M0, N0, K0, out, act, scales, bias, residual, pitch, lib.last_kernel_name())
    z = a @ b.T
    if scales:
        z = z * rs.cpu().double().numpy()[:, None] * cs.cpu().double().numpy()
    slack = np.abs(z) * 3 * U32
    if bias:
        z = z + bi.cpu().double().numpy()
        slack = slack + np.abs(z) * U32
    y = act64(z, act)
    # (No activation is steeper than 1.13.)
    slack = 1.13 * slack + act_slack(z, act)
    want = r64 + y
    half, tiny = HALF[out]
    slack = slack + np.abs(want) * U32
    got_buf = buf.cpu()
    got = at(got_buf, op, offset).double().numpy()
    off = np.abs(got - want) - (slack * (1 + half) + np.abs(want) * half + tiny)
    assert off.max() <= 0, (name, off.max(), np.unravel_index(off.argmax(), off.shape))
    at(got_buf, op, offset).copy_(at(before, op, offset))
    assert torch.equal(got_buf, before), name   # nothing else was written
    return name[-1]


TILES = [(S8, 16, 16, 16), (S8, 32, 16, 8), (S8, 1, 16, 16), (S8, 16, 16, 2), (S8, 8, 6, 4), (F8, 16, 16, 32), (F8, 1, 16, 16),
         (F16, 16, 16, 8), (F16, 1, 8, 16), (BF16, 16, 16, 8), (BF16, 16, 16, 2), (F32, 16, 16, 4), (F32, 16, 16, 1),
         (uk.MMT4D_TYPE_S16S16S32, 16, 16, 2), (uk.MMT4D_TYPE_S16S16S32, 4, 6, 3)]
MODES = [uk.KERNEL_MODE_AUTO, uk.KERNEL_MODE_GENERIC]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("type_,M0,N0,K0", TILES)
def test_epilogue_of_small_and_ragged_sizes(gpu, type_, M0, N0, K0, mode):
    """Every output type and activation, each part of the epilogue with and without, one row, one column,
    K of less than a step and ragged, loose rows at odd addresses, the residual apart and in place."""
    lib, _ = gpu
    lib.set_kernel_mode(mode)
    try:
        i = 0
        for rows, cols, k in [(1, 1, 5), (1, 70, 128), (3, 200, 1030), (17, 33, 64), (40, 150, 200), (70, 65, 512),
                              (130, 129, 96), (16, 500, 768)]:
            for out in OUTS:
                act = list(ACTS)[i % 5]
                run(lib, type_, rows, cols, k, M0, N0, K0, out, act, scales=i % 3 != 2, bias=i % 2 == 0,
                    residual=(None, "own", "in place", "own")[i % 4], pitch=(0, 3, 4)[i % 3], offset=(0, 1)[i % 2], seed=i)
                i += 1
    finally:
        lib.set_kernel_mode(uk.KERNEL_MODE_AUTO)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,M0,N0,K0", [(S8, 16, 16, 16), (F8, 16, 16, 32), (F16, 16, 16, 8), (BF16, 1, 16, 8),
                                            (S8, 32, 16, 8)])
@pytest.mark.parametrize("rows,cols,k", [
    (1, 4096, 4096), (16, 1040, 16384), (64, 3000, 1024), (200, 4096, 2048), (300, 300, 8192), (1000, 1501, 777),
    (2000, 40, 512), (40, 2000, 24576), (1030, 2050, 256), (2048, 4096, 128), (4100, 4200, 160), (4096, 8192, 64)])
def test_epilogue_of_layer_sizes(gpu, type_, M0, N0, K0, rows, cols, k):
    """The sizes at which the product's kernels change hands, from one row to several rounds of large blocks."""
    lib, _ = gpu
    i = rows + cols + k
    for j, (out, residual) in enumerate([("bf16", "own"), ("f32", "in place"), ("f16", None)]):
        run(lib, type_, rows, cols, k, M0, N0, K0, out, list(ACTS)[(i + j) % 5], bias=j != 1, scales=j != 2, residual=residual,
            seed=j)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,M0,N0,K0", [(S8, 16, 16, 16), (F8, 16, 16, 32), (BF16, 1, 16, 8), (F16, 24, 12, 8)])
def test_epilogue_with_rows_at_any_address(gpu, type_, M0, N0, K0):
    """Rows of whole groups of columns at odd pitches and offsets, in every kernel: what loads and stores
    16 bytes at once does so at any address of an element. Panels that do not divide a block (M0 = 24)."""
    lib, _ = gpu
    for i, (rows, cols, k) in enumerate([(1, 512, 1024), (40, 264, 100), (70, 1024, 512), (300, 512, 640), (520, 776, 320),
                                         (1024, 2048, 256), (2050, 2056, 200), (4096, 4096, 96)]):
        for j, (out, pitch, offset) in enumerate([("bf16", 1, 1), ("f32", 3, 1), ("f16", 8, 3)]):
            run(lib, type_, rows, cols, k, M0, N0, K0, out, list(ACTS)[(i + j) % 5], pitch=pitch, offset=offset,
                residual=("own", "in place", None)[(i + j) % 3], scales=i % 2 == 0, seed=i)


@pytest.mark.gpu
def test_epilogue_of_4_bit_weights(gpu):
    """s8 x s4, both in the kernel for few rows and on expanded weights, and the widened s16 x s8: types with a
    right-hand side of another width than the left-hand one's."""
    lib, _ = gpu
    rng = np.random.default_rng(3)
    for rows, cols, k, K0 in [(1, 512, 1024, 16), (40, 300, 512, 32), (70, 512, 448, 32), (600, 256, 512, 16), (5, 40, 96, 8)]:
        N1, K1 = -(-cols // 16), -(-k // K0)
        a = rng.integers(-8, 9, (rows, k))
        b = np.zeros((N1 * 16, K1 * K0), np.int64)
        b[:cols, :k] = rng.integers(-8, 8, (cols, k))
        t = b.reshape(N1, 16, K1, K0).transpose(0, 2, 1, 3).reshape(-1, 2) & 15
        rhs = torch.from_numpy((t[:, 0] | t[:, 1] << 4).astype(np.uint8)).cuda()
        full = np.zeros((rows, K1 * K0), np.int8)
        full[:, :k] = a
        lhs = torch.from_numpy(full).cuda()
        cs = torch.rand(cols, device="cuda") * 0.01
        res = torch.randn(rows, cols, device="cuda").to(torch.bfloat16)
        out = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
        lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, K1 * K0, rhs.data_ptr(), 0, K1 * 16 * K0, res.data_ptr(), 0, cols,
                                  out.data_ptr(), 0, cols, rows, cols, None, cs.data_ptr(), None, rows, N1, K1, 1, 16, K0,
                                  uk.MMT4D_TYPE_S8S4S32 | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION,
                                  uk.OUT_TYPE_BF16 | uk.ACTIVATION_RELU)
        lib.synchronize()
        z = (a @ b[:cols, :k].T) * cs.cpu().double().numpy()
        want = np.maximum(z, 0) + res.cpu().double().numpy()
        half, tiny = HALF["bf16"]
        off = np.abs(out.cpu().double().numpy() - want) - (np.abs(want) * half + (4 * U32 * np.abs(z) + 2 * U32 * np.abs(want)) * 2
                                                           + tiny)
        assert off.max() <= 0, (rows, cols, k, lib.last_kernel_name(), off.max())


@pytest.mark.gpu
def test_epilogue_of_a_product_over_no_k(gpu):
    """K == 0: what the epilogue makes of zeros."""
    lib, _ = gpu
    for out in OUTS:
        for residual in (None, "own"):
            run(lib, S8, 20, 33, 0, 16, 16, 16, out, "gelu", residual=residual)


@pytest.mark.gpu
def test_epilogue_passes_nan_scales_on(gpu):
    """A row whose scale is NaN (one without an 8-bit form) is NaN throughout, its neighbours are not."""
    lib, _ = gpu
    for act in ACTS:
        a = torch.ones(2, 4, 16, 16, dtype=torch.int8, device="cuda")
        rs = torch.ones(32, device="cuda")
        rs[5] = float("nan")
        out = torch.zeros(32, 48, device="cuda")
        b = torch.ones(3, 4, 16, 16, dtype=torch.int8, device="cuda")
        lib.mmt4d_epilogue_unpack(a.data_ptr(), 0, a.stride(0), b.data_ptr(), 0, b.stride(0), None, 0, 0, out.data_ptr(), 0, 48,
                                  32, 48, rs.data_ptr(), None, None, 2, 3, 4, 16, 16, 16, S8, uk.OUT_TYPE_F32 | ACTS[act])
        lib.synchronize()
        assert bool(out[5].isnan().all()) and not out[:5].isnan().any() and not out[6:].isnan().any(), act


@pytest.mark.gpu
def test_epilogue_in_a_captured_graph(gpu):
    """Captured and replayed on a side stream, with eager calls between, for the kernels that own a workspace
    outside a graph, too."""
    lib, _ = gpu
    s = torch.cuda.Stream()

    def capture(call):
        torch.cuda.synchronize()
        lib.set_stream(s.cuda_stream)
        lib.set_pointer_mode(uk.POINTER_MODE_DEVICE)
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                call()
            for _ in range(3):
                g.replay()
                torch.cuda.synchronize()
            call()
            torch.cuda.synchronize()   # (the replay runs on another stream, and writes the same matrix)
            g.replay()
            torch.cuda.synchronize()
        finally:
            lib.set_stream(None)
            lib.set_pointer_mode(uk.POINTER_MODE_AUTO)

    for type_, M0, N0, K0, rows, cols, k in [(S8, 16, 16, 16, 16, 512, 16384), (BF16, 16, 16, 2, 200, 300, 512),
                                             (F8, 16, 16, 32, 300, 300, 8192), (F32, 16, 16, 1, 40, 50, 60)]:
        for out in ("bf16", "f32"):
            run(lib, type_, rows, cols, k, M0, N0, K0, out, "silu", residual="own", capture=capture)


@pytest.mark.gpu
def test_epilogue_on_host_memory(gpu):
    lib, _ = gpu
    rng = np.random.default_rng(4)
    a = rng.integers(-9, 9, (20, 64)).astype(np.int8)
    b = rng.integers(-9, 9, (33, 64)).astype(np.int8)
    bias = rng.standard_normal(33).astype(np.float32)
    res = rng.standard_normal((20, 40)).astype(np.float32)
    rs = rng.random(20).astype(np.float32)
    want = np.maximum((a.astype(np.float64) @ b.T.astype(np.float64)) * rs[:, None] + bias, 0) + res[:, :33]
    for out in (np.full((20, 36), 7, np.float32), res):   # apart, and in place
        pitch = out.shape[1]
        lib.mmt4d_epilogue_unpack(a.ctypes.data, 0, 64, b.ctypes.data, 0, 64, res.ctypes.data, 0, 40, out.ctypes.data, 0, pitch,
                                  20, 33, rs.ctypes.data, None, bias.ctypes.data, 20, 33, 4, 1, 1, 16,
                                  S8 | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION, uk.OUT_TYPE_F32 | uk.ACTIVATION_RELU)
        assert np.abs(out[:, :33] - want).max() <= 8 * U32 * np.abs(want).max()
        if out is not res:
            assert (out[:, 33:] == 7).all()


def test_epilogue_refusals(lib):
    """Needs no device."""
    lib.raise_on_violation(True)

    def call(flags=S8, ep=uk.OUT_TYPE_BF16, rows=16, cols=16, M=1, stride=16, rstride=0, lhs=64, rhs=64, dst=64):
        lib.mmt4d_epilogue_unpack(lhs, 0, 0, rhs, 0, 0, None, 0, rstride, dst, 0, stride, rows, cols, None, None, None, M, 1,
                                  1, 16, 16, 16, flags, ep)

    for kw in [dict(flags=uk.MMT4D_TYPE_F16F16F16 | uk.MMT4D_SKIP_INTERMEDIATE_ROUNDINGS), dict(flags=0),
               dict(flags=S8 | uk.MMT4D_ACCUMULATE), dict(ep=0), dict(ep=uk.OUT_TYPE_S8), dict(ep=uk.OUT_TYPE_F8E4M3FN),
               dict(ep=uk.OUT_TYPE_F32 | 0x500), dict(ep=uk.OUT_TYPE_F32 | uk.IN_TYPE_F32), dict(ep=0x1010), dict(rows=17),
               dict(cols=17), dict(rows=-1), dict(stride=-16), dict(rstride=-1),
               dict(flags=uk.MMT4D_TYPE_S16S8S32), dict(stride=15), dict(stride=0), dict(lhs=None), dict(rhs=None),
               dict(dst=None)]:
        with pytest.raises(uk.ContractViolation):
            call(**kw)
    call(rows=0)
    call(cols=0)
    call(rows=0, M=0)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,K0", [(F8, 32), (F8, 16), (F16, 8), (BF16, 8)])
def test_f32_matrices_have_sums_in_f32(gpu, type_, K0):
    """Operands whose products spread over many binades: the sums keep f32. K additions, each rounded by
    up to 2^-24 of a sum that is no larger (in the root mean square) than the last one, and independently of
    one another, are off by sqrt(K) 2^-24 of it; by twice that if an instruction cuts off what others round.
    At K = 1000 that is 3.8e-6, where products that have lost their low bits are 1.3e-5 off."""
    lib, _ = gpu
    g = torch.Generator().manual_seed(5)
    names = set()
    for rows, cols, k in [(1, 300, 1000), (12, 109, 700), (40, 150, 333), (300, 300, 1000), (1000, 1100, 1000), (2100, 2100, 512)]:
        M0 = 1 if rows == 1 else 16
        M1, N1, K1 = -(-rows // M0), -(-cols // 16), -(-k // K0)

        def operand(n, t0, t1):
            full = torch.zeros(t1 * t0, K1 * K0)
            full[:n, :k] = 40 * torch.randn(n, k, generator=g)
            full = full.to(TORCH[type_])
            tiles = full.view(torch.int8 if type_ == F8 else torch.int16).view(t1, t0, K1, K0).transpose(1, 2).contiguous()
            return tiles.cuda(), full[:n].double()

        (lhs, a), (rhs, b) = operand(rows, M0, M1), operand(cols, 16, N1)
        out = torch.empty(rows, cols, device="cuda")
        lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(), None, 0, 0,
                                  out.data_ptr(), 0, cols, rows, cols, None, None, None, M1, N1, K1, M0, 16, K0, type_,
                                  uk.OUT_TYPE_F32)
        lib.synchronize()
        names.add(lib.last_kernel_name())
        want = a @ b.T
        off = ((out.cpu().double() - want).norm() / want.norm()).item()
        assert off <= 2 * k ** 0.5 * U32, (rows, cols, k, off, lib.last_kernel_name())
    assert len(names) >= 3, names


@pytest.mark.gpu
@pytest.mark.parametrize("type_,M0,K0", [(S8, 16, 16), (S8, 32, 8), (F8, 1, 32), (F16, 16, 8), (BF16, 1, 8)])
def test_slices_of_a_k_that_ends_inside_a_step(gpu, type_, M0, K0):
    """K in slices and what is left of it as one more, with a residual and without, row-major and at odd pitches."""
    lib, _ = gpu
    names = set()
    for rows, cols, k, residual, pitch in [(577, 716, 9001, "own", 0), (400, 1000, 12309, "in place", 3),
                                           (1000, 999, 16001, None, 1), (577, 716, 8968, "own", 5)]:
        for out in ("f32", "bf16"):
            names.add(run(lib, type_, rows, cols, k, M0, 16, K0, out, "silu", residual=residual, pitch=pitch, offset=pitch))
    assert any("kslices" in n for n in names), names


@pytest.mark.gpu
@pytest.mark.parametrize("type_,rows,cols,k", [(BF16, 700, 1700, 12309), (BF16, 700, 1700, 12288), (S8, 100, 300, 24700),
                                               (F8, 65, 65, 24576), (S8, 1700, 1300, 24600), (F8, 300, 300, 25695)])
def test_slices_of_a_long_k(gpu, type_, rows, cols, k):
    """From 24 KB of K on, few blocks and such as fill more than half of the units have K in slices."""
    lib, _ = gpu
    K0 = 8 if type_ == BF16 else 16
    names = set()
    for i, out in enumerate(("f32", "bf16")):
        names.add(run(lib, type_, rows, cols, k, 16, 16, K0, out, "silu", residual="own", pitch=i, offset=i))
    assert any("kslices" in n for n in names), names


@pytest.mark.gpu
@pytest.mark.parametrize("K0", [8, 4, 2, 1])
@pytest.mark.parametrize("residual", [None, "own", "in place"])
def test_f8_into_f32_keeps_f32_in_any_tile_rows(gpu, K0, residual):
    """test_f32_matrices_have_sums_in_f32 in tile rows under 16 bytes, from 2^24 multiply-adds on (fewer take the scalar
    kernel): the same tolerance, and two roundings of the residual's addition."""
    lib, _ = gpu
    g = torch.Generator().manual_seed(6)
    for rows, cols, k, M0 in [(300, 300, 1000, 16), (70, 700, 600, 8), (1000, 1100, 500, 16), (40, 900, 900, 1)]:
        M1, N1, K1 = -(-rows // M0), -(-cols // 16), -(-k // K0)

        def operand(n, t0, t1):
            full = torch.zeros(t1 * t0, K1 * K0)
            full[:n, :k] = 40 * torch.randn(n, k, generator=g)
            full = full.to(TORCH[F8])
            return full.view(torch.int8).view(t1, t0, K1, K0).transpose(1, 2).contiguous().cuda(), full[:n].double()

        (lhs, a), (rhs, b) = operand(rows, M0, M1), operand(cols, 16, N1)
        res = 1000 * torch.randn(rows, cols, generator=g)
        out = res.cuda() if residual == "in place" else torch.full((rows, cols), 7.0, device="cuda")
        own = out if residual == "in place" else res.cuda()
        lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(),
                                  own.data_ptr() if residual else None, 0, cols, out.data_ptr(), 0, cols, rows, cols, None,
                                  None, None, M1, N1, K1, M0, 16, K0, F8 | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION,
                                  uk.OUT_TYPE_F32)
        lib.synchronize()
        want = a[:, :k] @ b[:, :k].T
        total = want + (res.double() if residual else 0.0)
        off = ((out.cpu().double() - total).norm() / want.norm()).item()
        assert off <= (2 * k ** 0.5 + 2) * U32, (rows, cols, k, M0, off, lib.last_kernel_name())


def epilogue_of_bias(lib, x, rows, k, out, act, N0=16):
    """The matrix that a product of zeros and a bias of x make: activation(x) in every row."""
    n = x.numel()
    M1, N1, K1 = -(-rows // 16), -(-n // N0), -(-k // 16)
    lhs = torch.zeros(M1, K1, 16, 16, dtype=torch.int8, device="cuda")
    rhs = torch.zeros(N1, K1, N0, 16, dtype=torch.int8, device="cuda")
    dt, fo = OUTS[out]
    y = torch.full((rows, n), 7.0, dtype=dt, device="cuda")
    lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(), None, 0, 0, y.data_ptr(), 0,
                              n, rows, n, None, None, x.data_ptr(), M1, N1, K1, 16, N0, 16,
                              S8 | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION, fo | ACTS[act])
    lib.synchronize()
    return y


def gate_of(lib, x, act):
    y = torch.empty_like(x)
    n = x.numel()
    lib.gate_pack(x.data_ptr(), 0, n, None, 0, 0, y.data_ptr(), 0, n, None, 1, n, 1, n, 1, 1,
                  uk.IN_TYPE_F32 | uk.OUT_TYPE_F32 | ACTS[act])
    lib.synchronize()
    return y.view(1, n)


# rows, columns, K: few rows, few columns (operands change places), blocks of 32 to 256 rows, a width that ends inside
# eight columns, K in slices that another launch adds up.
BIAS_SIZES = [(1, 4096, 64), (700, 40, 64), (300, 2000, 64), (300, 2003, 64), (2300, 2048, 64), (4096, 4096, 64),
              (100, 304, 24576)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_sigmoids_into_f32_are_f32(gpu, act):
    """Into an f32 matrix a sigmoid is as close in its negative tail as near zero. With t the sigmoid's argument, in
    roundings of 2^-24: e^-t has 2 (the instruction's unit), 1 + e^-t 2, the reciprocal 2, the product with x 1; the
    remainder -t - hi ln 2 is kept, ln 2 itself being 2.8e-9 off, 0.05 roundings for each unit of t. GELU_TANH's t
    is four roundings of itself off. What a reciprocal of 2^126 and more would be is lost: |x| 2^-126."""
    lib, _ = gpu

    def check(y, x, name):
        v = x.cpu().double().numpy()
        t = np.abs(v if act == "silu" else v * (1.5957691216 + 0.0713548162726 * v * v))
        with np.errstate(over="ignore"):
            want = act64(v, act)
        slack = np.abs(want) * (8 + (0.05 if act == "silu" else 4.05) * t) * U32 + np.abs(v) * 2.0 ** -126 + 2.0 ** -149
        off = np.abs(y.cpu().double().numpy() - want) - slack
        assert off.max() <= 0, (name, act, off.max(), v[off.max(axis=0).argmax()])

    def values(n, seed):
        g = torch.Generator().manual_seed(seed)
        x = 4 * torch.randn(n, generator=g)
        x[::2] = -86 * torch.rand((n + 1) // 2, generator=g) if act == "silu" else -9 * torch.rand((n + 1) // 2, generator=g)
        return x.cuda()

    x = values(40000, 1)
    check(gate_of(lib, x, act), x, "gate_pack")
    names = set()
    for i, (rows, cols, k) in enumerate(BIAS_SIZES):
        for mode in MODES:
            lib.set_kernel_mode(mode)
            try:
                x = values(cols, i)
                check(epilogue_of_bias(lib, x, rows, k, "f32", act), x, (rows, cols, k, lib.last_kernel_name()))
                names.add(lib.last_kernel_name())
            finally:
                lib.set_kernel_mode(uk.KERNEL_MODE_AUTO)
            if k > 64:
                break   # (the scalar kernel: no K changes what it does behind its sums)
    assert len(names) >= 5, names


@pytest.mark.gpu
def test_gelu_is_its_fit(gpu):
    """GELU by e^(-s^2/2) t p(t), s = |x|. The constants as they are rounded give the tail s erfc(s / sqrt 2) / 2 to 7.5e-9
    and to 1.2e-7 s. Roundings of 2^-24 of the tail: 3 of t (its sum, the reciprocal's unit), of which the tail makes 2.8
    times as much; 3.2 of p, 1 each of three products, 2 of the exponential, 1.25 s^2 of its argument: 17 + 1.25 s^2.
    One of the result. Over 4096 neighbours those even out but for the units of the reciprocal and of the exponential,
    which may lean to one side: 8 of the tail, and the fit (one to 1.7e-7 does not pass). For positive x the rounding of
    x - tail does not even out either: x has no bits below its last, so neighbours whose tails differ by less than
    that bit (at x = 5 the tail is 1.4e-6, and all of 4096 results are x less the same multiple of 4.8e-7) are all
    rounded alike, by up to half of it: one rounding of the result more."""
    lib, _ = gpu
    windows = 96
    s = torch.linspace(0.02, 6.5, windows * 4096)
    for sign in (1.0, -1.0):
        x = (sign * s).cuda()
        got = [("gate_pack", gate_of(lib, x, "gelu"))]
        for lo in range(0, x.numel(), 32 * 4096):
            part = x[lo:lo + 32 * 4096]
            got.append((lo, epilogue_of_bias(lib, part, 1, 64, "f32", "gelu")))
        got = [got[0], ("epilogue", torch.cat([y for _, y in got[1:]], dim=1))]
        v = x.cpu().double().numpy()
        a = np.abs(v)
        want = act64(v, "gelu")
        tail = 0.5 * a * torch.special.erfc(torch.from_numpy(a * np.sqrt(0.5))).numpy()
        slack = np.minimum(7.5e-9, 1.2e-7 * a) + tail * (17 + 1.25 * a * a) * U32 + np.abs(want) * U32 + 2.0 ** -125
        for name, y in got:
            off = y.cpu().double().numpy()[0] - want
            assert (np.abs(off) - slack).max() <= 0, (name, sign, (np.abs(off) - slack).max())
            mean = np.abs(off.reshape(windows, -1).mean(axis=1))
            limit = 8 * U32 * tail + 4 * slack / 64 + (np.abs(want) * U32 if sign > 0 else 0.0)
            limit = 7.5e-9 + limit.reshape(windows, -1).mean(axis=1)
            assert (mean - limit).max() <= 0, (name, sign, mean.max())


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("spread", ["normal", "binades", "positive binades"])
def test_f8_into_16_bits_is_off_by_what_its_instructions_lose(gpu, out, spread):
    """The 8-bit float instructions add products eight by eight and lose what lies 13 binades and more below the largest of
    the eight: 7 * 2^-13 of it at most, so 2^-10 of the sum of magnitudes; for normal operands 2^-15 of the root mean
    square at most. Seen behind a residual that cancels the product, so that the matrix's own roundings are small."""
    lib, _ = gpu
    g = torch.Generator().manual_seed(8)
    dt, fo = OUTS[out]
    half, tiny = HALF[out]
    for rows, cols, k, M0 in [(1, 64, 512, 1), (16, 300, 4096, 16), (300, 300, 1024, 16), (300, 300, 24608, 16),
                              (2100, 2100, 512, 16)]:
        def operand(n, t0):
            v = torch.exp2(14 * torch.rand(n, k, generator=g) - 6).clamp(max=448)
            if spread == "normal":
                v = 40 * torch.randn(n, k, generator=g)
            elif spread == "binades":
                v = v * torch.randn(n, k, generator=g).sign()
            t1 = -(-n // t0)
            full = torch.zeros(t1 * t0, k)
            full[:n] = v
            full = full.to(TORCH[F8])
            return full.view(torch.int8).view(t1, t0, k // 32, 32).transpose(1, 2).contiguous().cuda(), full[:n].double()

        (lhs, a), (rhs, b) = operand(rows, M0), operand(cols, 16)
        z, sums = a @ b.T, a.abs() @ b.abs().T
        scale = 2.0 ** -np.ceil(np.log2(sums.max().item() / 16384))   # (a power of two: exact)
        z, sums = z * scale, sums * scale
        res = (-z).to(dt)
        rs = torch.full((rows,), scale, device="cuda")
        res_gpu, y = res.cuda(), torch.empty(rows, cols, dtype=dt, device="cuda")
        lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(), res_gpu.data_ptr(), 0,
                                  cols, y.data_ptr(), 0, cols, rows, cols, rs.data_ptr(), None, None, lhs.shape[0], rhs.shape[0],
                                  k // 32, M0, 16, 32, F8, fo)
        lib.synchronize()
        want = z + res.double()
        off = (y.cpu().double() - want).abs()
        # (2^-24 a step of the sum and one for the factor; the matrix's rounding)
        slack = sums * (2.0 ** -10 + (k / 32 + 2) * U32)
        assert ((off - (slack + (want.abs() + slack) * half + tiny)).max().item()) <= 0, (rows, cols, k, lib.last_kernel_name())
        if spread == "normal":
            rms = lambda t: t.pow(2).mean().sqrt().item()  # noqa: E731
            assert rms(off) <= 2.0 ** -15 * rms(z) + half * rms(want) + tiny, (rows, cols, k, rms(off) / rms(z))


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [None, "own", "in place"])
@pytest.mark.parametrize("type_,M0,N0,K0,rows,cols,k", [
    (S8, 16, 16, 16, 16, 512, 16384), (S8, 32, 16, 8, 40, 264, 512), (BF16, 16, 16, 2, 200, 300, 512),
    (F16, 16, 16, 8, 520, 776, 320), (F8, 16, 16, 32, 300, 300, 8192), (F8, 1, 16, 32, 1, 1000, 4096),
    (F8, 16, 16, 8, 100, 120, 256), (F32, 16, 16, 1, 40, 50, 60), (S8, 16, 16, 16, 2050, 2056, 256)])
def test_every_replay_of_a_captured_epilogue_writes_its_matrix(gpu, type_, M0, N0, K0, rows, cols, k, residual):
    """The matrix is made unusable before each replay (in place: the residual put back), and compared after it. Small
    integers throughout: sums are exact, results are roundings of them. Eager calls between the replays."""
    lib, _ = gpu
    rng = np.random.default_rng(rows)
    M1, N1, K1 = -(-rows // M0), -(-cols // N0), -(-k // K0)
    a, b = rng.integers(-4, 5, (rows, k)).astype(np.float64), rng.integers(-4, 5, (cols, k)).astype(np.float64)
    lhs, rhs = tiled(a, M0, K0, M1, K1, TORCH[type_]), tiled(b, N0, K0, N1, K1, TORCH[type_])
    s = torch.cuda.Stream()
    for out in ("bf16", "f32"):
        dt, fo = OUTS[out]
        res = torch.from_numpy(rng.integers(-64, 65, (rows, cols)).astype(np.float32)).to(dt).cuda()
        want = torch.from_numpy(np.maximum(a @ b.T, 0)).cuda() + (res.double() if residual else 0.0)
        want = want.to(torch.float32).to(dt)
        buf = torch.empty(rows, cols, dtype=dt, device="cuda")
        from_ = None if residual is None else (buf if residual == "in place" else res).data_ptr()

        def call():
            lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(), from_, 0, cols,
                                      buf.data_ptr(), 0, cols, rows, cols, None, None, None, M1, N1, K1, M0, N0, K0,
                                      type_ | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION, fo | uk.ACTIVATION_RELU)

        def checked(run_once, what):
            if residual == "in place":
                buf.copy_(res)
            else:
                buf.fill_(float("nan"))
            torch.cuda.synchronize()
            run_once()
            torch.cuda.synchronize()
            assert torch.equal(buf, want), (what, out, lib.last_kernel_name(), (buf.double() - want.double()).abs().max().item())

        torch.cuda.synchronize()
        lib.set_stream(s.cuda_stream)
        lib.set_pointer_mode(uk.POINTER_MODE_DEVICE)
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                call()
            for i in range(3):
                checked(g.replay, "replay %d" % i)
                checked(call, "eager %d" % i)
        finally:
            lib.set_stream(None)
            lib.set_pointer_mode(uk.POINTER_MODE_AUTO)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1792, 1664), (1920, 1280)])
def test_slices_keep_the_memory_that_the_header_names(gpu, rows, cols):
    """182 and 150 blocks of 64 KB with K in slices of whole steps, and its end as one more: 64 MB of sums, and the workspace's
    counters. (At 24 KB of K the costs are 115 us for four slices of 182 blocks, 96 for three of 150, where five, from
    42 KB on, would keep as much: 60 MB.)"""
    lib, _ = gpu
    lib.release_workspaces()
    name = run(lib, S8, rows, cols, 24603, 16, 16, 16, "bf16", "none", residual="own")
    assert "kslices" in name and lib.last_k_slices() >= 3, (name, lib.last_k_slices())
    kept = lib.workspace_bytes()
    assert 0 < kept <= (64 << 20) + (64 << 10), kept
    lib.release_workspaces()
    assert lib.workspace_bytes() == 0


def exact_epilogue(lib, type_, rows, cols, k, M0, N0, K0, out, *, residual, panels=(0, 0), on="cuda", seed=0):
    """A call whose results are exact: small integers, row scales of powers of two, RELU. `residual`: None, "own", "in place"
    or "one row" (a stride of 0). `panels`: tiles beyond those that the matrix needs, which hold what must not matter."""
    rng = np.random.default_rng(seed)
    M1, N1, K1 = -(-rows // M0) + panels[0], -(-cols // N0) + panels[1], -(-k // K0)
    a, b = rng.integers(-4, 5, (rows, k)).astype(np.float64), rng.integers(-4, 5, (cols, k)).astype(np.float64)
    lhs, rhs = tiled(a, M0, K0, M1, K1, TORCH[type_]).to(on), tiled(b, N0, K0, N1, K1, TORCH[type_]).to(on)
    dt, fo = OUTS[out]
    rs = torch.exp2(torch.from_numpy(rng.integers(-2, 3, rows)).float())
    n_res = 1 if residual == "one row" else rows
    res = torch.from_numpy(rng.integers(-64, 65, (n_res, cols)).astype(np.float32)).to(dt)
    want = torch.from_numpy(np.maximum(a @ b.T, 0)) * rs.double()[:, None] + (res.double() if residual else 0.0)
    want = want.float().to(dt)
    buf = torch.full((rows + 1, cols + 3), 7.0, dtype=dt)
    if residual == "in place":
        buf[:rows, :cols] = res
    before = buf.clone()
    buf, rs_on, res_on = buf.to(on), rs.to(on), res.to(on)
    from_, stride = {None: (None, 0), "own": (res_on, cols), "one row": (res_on, 0), "in place": (buf, cols + 3)}[residual]
    lib.mmt4d_epilogue_unpack(lhs.data_ptr(), 0, lhs[0].numel(), rhs.data_ptr(), 0, rhs[0].numel(),
                              from_.data_ptr() if from_ is not None else None, 0, stride, buf.data_ptr(), 0, cols + 3, rows,
                              cols, rs_on.data_ptr(), None, None, M1, N1, K1, M0, N0, K0,
                              type_ | uk.MMT4D_ALLOW_GENERIC_FALLBACK_TILE_FUNCTION, fo | uk.ACTIVATION_RELU)
    name = (type_, rows, cols, k, M0, N0, K0, out, residual, panels, on, lib.last_kernel_name())
    lib.synchronize()
    got = buf.cpu()
    assert torch.equal(got[:rows, :cols], want), name
    got[:rows, :cols] = before[:rows, :cols]
    assert torch.equal(got, before), name
    return name[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("type_,M0,N0,K0", [(F32, 16, 16, 4), (F32, 1, 16, 1), (BF16, 16, 16, 2), (F8, 16, 16, 8)])
@pytest.mark.parametrize("residual", [None, "own", "in place", "one row"])
def test_a_product_apart_in_several_rounds_of_rows(gpu, type_, M0, N0, K0, residual):
    """Products of more than 64 MB of f32 in front of an epilogue of their own: rounds of rows, each with its scales and
    its rows of the residual."""
    lib, _ = gpu
    for out in ("f32", "bf16"):
        exact_epilogue(lib, type_, 4501, 4099, 24, M0, N0, K0, out, residual=residual)


@pytest.mark.gpu
@pytest.mark.parametrize("type_,M0,N0,K0", [(S8, 16, 16, 16), (S8, 1, 16, 16), (S8, 32, 16, 8), (F8, 16, 16, 32), (F8, 16, 16, 4),
                                            (BF16, 16, 16, 8), (F16, 24, 12, 8), (F32, 16, 16, 4)])
def test_tiles_beyond_the_matrix_and_a_residual_of_one_row(gpu, type_, M0, N0, K0):
    """More tiles than the matrix has rows and columns for, from one row to several rounds of blocks and K in slices; a
    residual whose rows are all the same one."""
    lib, _ = gpu
    for i, (rows, cols, k) in enumerate([(1, 300, 256), (3, 70, 1030), (40, 33, 512), (300, 500, 200), (700, 1500, 320),
                                         (130, 300, 24703), (2050, 2060, 96)]):
        for out, residual in (("bf16", "one row"), ("f32", "in place"), ("f32", "one row")):
            exact_epilogue(lib, type_, rows, cols, k, M0, N0, K0, out, residual=residual, panels=(i % 3, (i + 1) % 4), seed=i)


@pytest.mark.gpu
def test_epilogue_on_host_memory_with_a_residual_of_one_row(gpu):
    lib, _ = gpu
    for out in ("f32", "bf16"):
        for residual in ("one row", "in place", "own", None):
            exact_epilogue(lib, S8, 37, 50, 96, 16, 16, 16, out, residual=residual, panels=(1, 1), on="cpu")
