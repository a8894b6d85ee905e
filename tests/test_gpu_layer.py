"""The calls between two products together, as a layer runs them: residual
addition and norm into tiles, the gate and up projections, their activation into
tiles, the down projection onto the residual stream. Each step is checked
against its formula in 64 bits on what the step before it has left, eager and
replayed from a graph."""
import numpy as np
import pytest
import torch

from iree_amd import ukernel as uk
from test_gpu_row_ops import HALF, LARGEST, OUTS, U32, act64, act_slack, check_rows, f8_value, norm_reference, tiles_to_matrix

# weights' type -> (mmt4d type, N0, K0, the type of the steps' tiles)
KINDS = {"s8": (uk.MMT4D_TYPE_S8S8S32, 16, 16, "s8"), "s8 8-byte rows": (uk.MMT4D_TYPE_S8S8S32, 16, 8, "s8"),
         "f8": (uk.MMT4D_TYPE_F8E4M3FNF8E4M3FNF32, 16, 32, "f8"), "bf16": (uk.MMT4D_TYPE_BF16BF16F32, 16, 8, "bf16")}


class Layer:
    def __init__(self, kind, rows, d, hidden, M0, seed):
        self.type_, self.N0, self.K0, self.tout = KINDS[kind]
        self.rows, self.d, self.hidden, self.M0 = rows, d, hidden, M0
        rng = np.random.default_rng(seed)
        bf = lambda a: torch.from_numpy(a).float().to(torch.bfloat16).cuda()  # noqa: E731
        self.x = bf(2 * rng.standard_normal((rows, d)))
        self.delta = bf(rng.standard_normal((rows, d)))
        self.norm_weight = bf(1 + 0.1 * rng.standard_normal(d))
        self.stream = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda")
        self.w1, self.s1 = self.weights(rng, 2 * hidden, d)
        self.w2, self.s2 = self.weights(rng, d, hidden)
        self.bias = torch.from_numpy(0.1 * rng.standard_normal(2 * hidden)).float().cuda()
        self.tiles1, self.scale1 = self.tiles(d)
        self.tiles2, self.scale2 = self.tiles(hidden)
        self.both = torch.empty(rows, 2 * hidden, dtype=torch.bfloat16, device="cuda")

    def tiles(self, k):
        dt = OUTS[self.tout][0] if self.tout in OUTS else torch.bfloat16
        t = torch.zeros(-(-self.rows // self.M0), -(-k // self.K0), self.M0, self.K0, dtype=dt, device="cuda")
        return t, torch.zeros(self.rows, device="cuda") if self.tout in LARGEST else None

    def weights(self, rng, n, k):
        """n x k weights in tiles, and a scale a column of the result."""
        n1, k1 = -(-n // self.N0), -(-k // self.K0)
        w = np.zeros((n1 * self.N0, k1 * self.K0))
        v = rng.standard_normal((n, k))
        w[:n, :k] = np.rint(v * 40).clip(-127, 127) if self.tout == "s8" else v * 60 if self.tout == "f8" else v / np.sqrt(k)
        t = torch.from_numpy(w).float().view(n1, self.N0, k1, self.K0).transpose(1, 2).contiguous()
        t = t.to({"s8": torch.int8, "f8": torch.float8_e4m3fn, "bf16": torch.bfloat16}[self.tout]).cuda()
        width = {"s8": 40.0, "f8": 60.0}.get(self.tout)
        s = torch.from_numpy((0.5 + rng.random(n)) / (width * np.sqrt(k))).float().cuda() if width else None
        return t, s

    def product(self, lib, tiles, scale, w, cols, out, out_flags, bias, residual):
        n = out.shape[1]
        lib.mmt4d_epilogue_unpack(
            tiles.data_ptr(), 0, tiles[0].numel(), w.data_ptr(), 0, w[0].numel(), residual.data_ptr() if residual is not None else
            None, 0, n, out.data_ptr(), 0, n, self.rows, n, scale.data_ptr() if scale is not None else None,
            cols.data_ptr() if cols is not None else None, bias.data_ptr() if bias is not None else None, tiles.shape[0],
            w.shape[0], tiles.shape[1], self.M0, self.N0, self.K0, self.type_, out_flags)

    def run(self, lib):
        out = OUTS[self.tout][1] if self.tout in OUTS else uk.OUT_TYPE_BF16
        t = self.tiles1
        lib.rmsnorm_pack(self.x.data_ptr(), 0, self.d, self.delta.data_ptr(), 0, self.d, self.stream.data_ptr(), 0, self.d,
                         self.norm_weight.data_ptr(), 1e-5, t.data_ptr(), 0, t.stride(0), self.scale1.data_ptr()
                         if self.scale1 is not None else None, self.rows, self.d, *t.shape, uk.IN_TYPE_BF16 | out)
        self.product(lib, t, self.scale1, self.w1, self.s1, self.both, uk.OUT_TYPE_BF16, self.bias, None)
        self.after_norm = self.stream.clone() if not torch.cuda.is_current_stream_capturing() else None
        t = self.tiles2
        lib.gate_pack(self.both.data_ptr(), 0, 2 * self.hidden, self.both.data_ptr(), self.hidden, 2 * self.hidden, t.data_ptr(),
                      0, t.stride(0), self.scale2.data_ptr() if self.scale2 is not None else None, self.rows, self.hidden,
                      *t.shape, uk.IN_TYPE_BF16 | out | uk.ACTIVATION_SILU)
        self.product(lib, t, self.scale2, self.w2, self.s2, self.stream, uk.OUT_TYPE_BF16, None, self.stream)

    def outputs(self):
        return [t for t in (self.tiles1, self.scale1, self.both, self.tiles2, self.scale2, self.stream) if t is not None]


def values(t):
    return f8_value(t.cpu()) if t.dtype == torch.uint8 else t.cpu().double().numpy()


def check_product(layer, tiles, scale, w, cols, bias, residual, got, name):
    """Float operands: a sum of k products in f32, 2^-16 of the sum of their magnitudes at most (matrix
    instructions of 8-bit floats align what they add to their largest term; the others are closer)."""
    k = w.shape[1] * w.shape[3]
    a = tiles_to_matrix(values(tiles))[:layer.rows]
    b = tiles_to_matrix(w.cpu().double().numpy())[:got.shape[1]]
    factor = (scale.cpu().double().numpy()[:, None] if scale is not None else 1.0) * (cols.cpu().double().numpy() if cols is not
                                                                                     None else 1.0)
    z = a @ b.T * factor
    slack = np.abs(z) * 4 * U32
    if layer.tout != "s8":
        slack = slack + np.abs(a) @ np.abs(b).T * np.abs(factor) * (2.0 ** -16 if layer.tout == "f8" else min(k, 64) * U32)
    want = z + (bias.cpu().double().numpy() if bias is not None else 0.0)
    want = want + (residual.cpu().double().numpy() if residual is not None else 0.0)
    half, tiny = HALF["bf16"]
    off = np.abs(got.cpu().double().numpy() - want) - ((slack + 2 * U32 * np.abs(want)) * (1 + half) + np.abs(want) * half + tiny)
    assert off.max() <= 0, (name, off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows,d,hidden,M0", [(1, 512, 1408, 1), (16, 512, 1408, 32), (5, 500, 1001, 16), (200, 640, 1536, 16),
                                              (300, 1024, 2816, 16)])
def test_a_gated_layer(gpu, kind, rows, d, hidden, M0):
    lib, _ = gpu
    if kind == "s8 8-byte rows" and M0 == 1:
        M0 = 2
    layer = Layer(kind, rows, d, hidden, M0, rows)
    name = (kind, rows)
    torch.cuda.synchronize()
    layer.run(lib)
    lib.synchronize()
    h, y, slack = norm_reference(layer.x.cpu().double().numpy(), layer.delta.cpu().double().numpy(),
                                 layer.norm_weight.cpu().double().numpy(), 1e-5, d)
    half, tiny = HALF["bf16"]
    assert np.all(np.abs(layer.after_norm.cpu().double().numpy() - h) <= np.abs(h) * (half + 2 * U32) + tiny), name
    sc = lambda t: t.cpu().double().numpy() if t is not None else None  # noqa: E731
    check_rows(y, slack, "bf16", layer.tout, values(layer.tiles1), sc(layer.scale1), rows, d, name)
    check_product(layer, layer.tiles1, layer.scale1, layer.w1, layer.s1, layer.bias, None, layer.both, name)
    both = layer.both.cpu().double().numpy()
    gate, up = both[:, :hidden], both[:, hidden:]
    check_rows(act64(gate, "silu") * up, act_slack(gate, "silu") * np.abs(up) + np.abs(act64(gate, "silu") * up) * U32, "bf16",
               layer.tout, values(layer.tiles2), sc(layer.scale2), rows, hidden, name)
    check_product(layer, layer.tiles2, layer.scale2, layer.w2, layer.s2, None, layer.after_norm, layer.stream, name)

    # The same from a graph, several times, with eager runs between.
    eager = [t.clone() for t in layer.outputs()]
    s = torch.cuda.Stream()
    lib.set_pointer_mode(uk.POINTER_MODE_DEVICE)
    lib.set_stream(s.cuda_stream)
    try:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            layer.run(lib)
        for i in range(3):
            for t in layer.outputs():
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            first = [t.clone() for t in layer.outputs()]
            if i == 0:
                replayed = first
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(replayed, first)), name
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                layer.run(lib)
            torch.cuda.synchronize()
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(eager, layer.outputs())), name
        # (A graph's products run unsplit: other roundings of their sums, integers excepted.)
        if layer.tout == "s8":
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(eager, replayed)), name
    finally:
        lib.set_stream(None)
        lib.set_pointer_mode(uk.POINTER_MODE_AUTO)


@pytest.mark.gpu
def test_layers_of_two_threads_at_once(gpu):
    """Two threads with a stream each run layers side by side; results as alone."""
    import threading
    lib, _ = gpu
    layers = [Layer(kind, 40, 512, 1408, 16, 7) for kind in ("s8", "f8")]
    alone = []
    for layer in layers:
        layer.run(lib)
        lib.synchronize()
        alone.append([t.clone() for t in layer.outputs()])
    torch.cuda.synchronize()
    problems = []

    def work(layer, want):
        try:
            s = torch.cuda.Stream()
            lib.lib.iree_uk_amd_set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                for _ in range(20):
                    layer.run(lib)
            s.synchronize()
            if not all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, layer.outputs())):
                problems.append("other results")
        except Exception as e:   # noqa: BLE001
            problems.append(repr(e))

    threads = [threading.Thread(target=work, args=p) for p in zip(layers, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not problems, problems
