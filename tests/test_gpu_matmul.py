"""Products with packed weights on the GPU against 64-bit products of the oracle's decoded weights (tests/matmul_ref.py
derives the bounds)."""
import numpy as np
import pytest

import matmul_ref as ref
from util import same_bits, same_bits16

pytestmark = pytest.mark.gpu

TYPES = [1, 30, 2, 3, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 20, 23]
KIND = {"f32": 0, "f16": 1, "bf16": 30}
SENTINEL = 77.0


def dtype(kind):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def weights(ty, rows, cols, seed):
    import gguf_amd as g
    from gguf_amd import synth
    return synth.random_blocks(ty, rows * cols // g.block_elems(ty), seed)


def activations(tokens, cols, kind, seed, stride=None):
    """A device tensor [tokens, cols] inside a buffer of `stride` elements a row, and its values in 64 bits."""
    import torch
    v = np.random.default_rng(seed).standard_normal((tokens, stride or cols)).astype(np.float32)
    x = torch.from_numpy(v).cuda().to(dtype(kind))[:, :cols]
    return x, x.double().cpu().numpy()


def output(tokens, rows, kind, stride=None):
    """A buffer of sentinels with a row to spare before and behind, and the view that is written."""
    import torch
    buf = torch.full((tokens + 2, stride or rows), SENTINEL, dtype=dtype(kind), device="cuda")
    return buf, buf[1:tokens + 1, :rows]


def untouched(buf, tokens, rows):
    b = buf.float().cpu().numpy()
    return bool((b[0] == SENTINEL).all() and (b[-1] == SENTINEL).all() and (b[1:-1, rows:] == SENTINEL).all())


def on_device(packed, offset=0):
    """The bytes on the device, `offset` bytes off an aligned address."""
    import torch
    t = torch.zeros(packed.size + offset, dtype=torch.uint8, device="cuda")
    t[offset:] = torch.from_numpy(packed).cuda()
    return t[offset:]


def run_matvec(oracle, ty, rows, cols, tokens, xk, yk, seed, x_stride=None, y_stride=None, offset=0):
    import gguf_amd as g
    import torch
    p = weights(ty, rows, cols, seed)
    x, x64 = activations(tokens, cols, xk, seed + 1, x_stride)
    buf, y = output(tokens, rows, yk, y_stride)
    g.matvec(ty, y, on_device(p, offset), x)
    torch.cuda.synchronize()
    want, bound = ref.product(*ref.decode(oracle, ty, p, rows, cols), x64)
    got = y.float().cpu().numpy()
    assert ref.outside(got, want, bound, yk) == 0, (np.abs(got - want).max(), np.unravel_index(np.argmax(np.abs(got - want) - bound), got.shape))
    assert untouched(buf, tokens, rows)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("rows,blocks,tokens,xk,yk", [
    (1, 1, 1, "f32", "f32"), (3, 2, 1, "bf16", "f32"), (4, 3, 1, "f16", "f32"), (5, 7, 2, "f32", "bf16"), (67, 8, 1, "bf16", "bf16"),
    (33, 5, 3, "f16", "f16"), (130, 16, 4, "f32", "f32"), (9, 33, 5, "bf16", "f32"), (257, 4, 16, "f16", "f32"), (64, 9, 17, "f32", "f16"),
    (31, 17, 33, "bf16", "f16")])
def test_matvec(oracle, ty, rows, blocks, tokens, xk, yk):
    cols = blocks * (oracle.block_elems(ty) if ty not in (1, 30) else 1)
    run_matvec(oracle, ty, rows, cols, tokens, xk, yk, 100 * ty + rows)


@pytest.mark.parametrize("ty", [2, 3, 8, 20, 1, 30])
@pytest.mark.parametrize("cols", [32, 64, 96, 480, 512, 544, 1024, 1184, 2048, 2080, 8224])
@pytest.mark.parametrize("xk", ["f32", "bf16"])
def test_matvec_row_lengths(oracle, ty, cols, xk):
    """Rows that end inside a lane's, a wave's or a workgroup's share."""
    run_matvec(oracle, ty, 21, cols, 1, xk, "f32", cols + ty)
    run_matvec(oracle, ty, 6, cols, 6, xk, "f32", cols + ty + 1)


@pytest.mark.parametrize("ty", [1, 30])
@pytest.mark.parametrize("cols", [1, 3, 7, 33, 63, 65, 1001])
def test_matvec_float_weights_odd_lengths(oracle, ty, cols):
    for offset in (0, 1, 2):
        run_matvec(oracle, ty, 19, cols, 3, "f32", "f32", cols, offset=offset)


@pytest.mark.parametrize("ty", TYPES)
def test_matvec_long_rows(oracle, ty):
    """Rows whose activations do not fit in a workgroup's shared memory at once."""
    cols = 28672 if ty not in (1, 30) else 28671
    for tokens, xk in ((1, "f32"), (4, "bf16"), (7, "f32"), (16, "f16")):
        run_matvec(oracle, ty, 37, cols, tokens, xk, "f32", 7 * ty + tokens)


@pytest.mark.parametrize("ty", [2, 8, 10, 12, 14, 15, 23, 1])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 8, 14])
def test_matvec_alignment_and_strides(oracle, ty, offset):
    """Packed bytes at any address; rows of x and y inside wider buffers, at odd distances too."""
    run_matvec(oracle, ty, 45, 2304, 3, "bf16", "f16", offset + ty, x_stride=2304 + 8 * offset + 1, y_stride=45 + offset, offset=offset)
    run_matvec(oracle, ty, 45, 768, 1, "f32", "f32", offset + ty, x_stride=769, y_stride=46, offset=offset)
    run_matvec(oracle, ty, 18, 768, 9, "f16", "bf16", offset + ty, x_stride=771 + offset, y_stride=21, offset=offset)


def test_matvec_one_row_for_all_tokens_vectors_and_empty(oracle):
    import torch
    import gguf_amd as g
    p = weights(12, 40, 512, 1)
    w = on_device(p)
    x, x64 = activations(1, 512, "f32", 2)
    want, bound = ref.product(*ref.decode(oracle, 12, p, 40, 512), x64)
    y = torch.empty(6, 40, device="cuda")
    g.matvec(12, y, w, x.expand(6, 512))                        # stride 0 between the tokens
    v = torch.empty(40, device="cuda")
    g.Q4K.matvec(v, w, x[0])                                    # vectors
    torch.cuda.synchronize()
    for t in range(6):
        assert ref.outside(y[t:t + 1].cpu().numpy(), want, bound, "f32") == 0
    assert ref.outside(v[None].cpu().numpy(), want, bound, "f32") == 0
    z = torch.full((3, 5), 9.0, device="cuda")
    g.matvec(2, z, torch.empty(0, dtype=torch.uint8, device="cuda"), torch.empty(3, 0, device="cuda"))
    g.matvec(2, torch.empty(0, 5, device="cuda"), torch.zeros(5 * 18, dtype=torch.uint8, device="cuda"), torch.empty(0, 32, device="cuda"))
    torch.cuda.synchronize()
    assert bool((z == 0).all())                                 # a sum of nothing


@pytest.mark.parametrize("xk", ["f32", "f16", "bf16"])
def test_matvec_values_of_every_size(oracle, xk):
    """Activations from the type's smallest numbers to large ones, zeros among them, in one row."""
    import torch
    import gguf_amd as g
    for ty in (2, 12, 14, 20, 1):
        rows, cols = 24, 1024
        p = weights(ty, rows, cols, ty)
        rng = np.random.default_rng(ty)
        span = {"f32": (-120, 60), "f16": (-24, 10), "bf16": (-120, 60)}[xk]
        v = rng.standard_normal((2, cols)) * 2.0 ** rng.integers(*span, (2, cols))
        v[:, ::7] = 0.0
        v[1, 256:] *= 2.0 ** -12 if xk == "f16" else 2.0 ** -20
        x = torch.from_numpy(v.astype(np.float32)).cuda().to(dtype(xk))
        y = torch.empty(2, rows, device="cuda")
        g.matvec(ty, y, on_device(p), x)
        torch.cuda.synchronize()
        want, bound = ref.product(*ref.decode(oracle, ty, p, rows, cols), x.double().cpu().numpy())
        assert ref.outside(y.cpu().numpy(), want, bound, "f32") == 0


def test_matvec_non_finite_stays_where_it_is(oracle):
    """A token with an infinity or a NaN, and a row with a non-finite scale, leave the others alone."""
    import torch
    import gguf_amd as g
    for ty, tokens in ((2, 3), (12, 4), (14, 5), (1, 6), (8, 16), (30, 1)):
        rows, cols = 37, 1536
        p = weights(ty, rows, cols, ty)
        bb, be = g.block_bytes(ty), g.block_elems(ty)
        at = {14: 208}.get(ty, 0)
        row = 5 * (cols // be) * bb + at
        p[row:row + 2] = (0x80, 0x7F) if ty == 30 else (0x00, 0x7C)              # +inf
        x, _ = activations(tokens, cols, "f32", 3)
        x = x.clone()
        if tokens > 2:
            x[1, 700] = float("inf")
            x[2, 3] = float("nan")
        y = torch.empty(tokens, rows, device="cuda")
        g.matvec(ty, y, on_device(p), x)
        torch.cuda.synchronize()
        got = y.cpu().numpy()
        clean = [t for t in range(tokens) if tokens <= 2 or t not in (1, 2)]
        q = p.copy()
        q[row:row + 2] = 0
        want, bound = ref.product(*ref.decode(oracle, ty, q, rows, cols), x[clean].double().cpu().numpy())
        others = [r for r in range(rows) if r != 5]
        assert ref.outside(got[clean][:, others], want[:, others], bound[:, others], "f32") == 0
        assert not np.isfinite(got[:, 5]).any()
        if tokens > 2:
            assert np.isnan(got[2]).all()
            assert not np.isfinite(got[1]).any() or ty in (1, 30)


def test_matvec_repeats_bit_for_bit_and_replays_from_a_graph(oracle):
    """The same inputs give the same bits, eagerly, on another stream and from a graph that is replayed with new inputs."""
    import torch
    import gguf_amd as g
    cases = []
    for ty, rows, cols, tokens, xk in ((12, 600, 2048, 1, "bf16"), (14, 200, 4096, 3, "f32"), (2, 96, 1184, 16, "f16"), (1, 50, 333, 2, "f32")):
        p = weights(ty, rows, cols, ty)
        x, _ = activations(tokens, cols, xk, ty)
        cases.append((ty, on_device(p), x.contiguous(), torch.empty(tokens, rows, device="cuda")))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        for ty, w, x, y in cases:
            g.matvec(ty, y, w, x)
    torch.cuda.current_stream().wait_stream(side)
    first = [y.clone() for *_, y in cases]
    with torch.cuda.graph(graph):
        for ty, w, x, y in cases:
            g.matvec(ty, y, w, x)
    for rep in range(4):
        if rep:
            for i, (ty, w, x, y) in enumerate(cases):
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * rep + i)).to(x.dtype))
        for *_, y in cases:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, (ty, w, x, y) in enumerate(cases):
            again = torch.empty_like(y)
            g.matvec(ty, again, w, x)
            torch.cuda.synchronize()
            assert torch.equal(again, y)
            if rep == 0:
                assert torch.equal(first[i], y)


def test_two_streams_at_once(oracle):
    import torch
    import gguf_amd as g
    p = weights(12, 3000, 4096, 1)
    w = on_device(p)
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [activations(1, 4096, k, i)[0] for i, k in enumerate(("bf16", "f32"))]
    torch.cuda.synchronize()
    outs = [[torch.empty(1, 3000, device="cuda") for _ in range(8)] for _ in streams]
    for k in range(8):
        for s, x, o in zip(streams, xs, outs):
            g.matvec(12, o[k], w, x, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for x, o in zip(xs, outs):
        alone = torch.empty(1, 3000, device="cuda")
        g.matvec(12, alone, w, x)
        for y in o:
            assert torch.equal(y, alone)


def test_matrix_beyond_32_bit_offsets(oracle):
    """A packed matrix of more than 4 GiB: its last rows."""
    import torch
    import gguf_amd as g
    cols, bb = 8192, 34 * 8192 // 32
    rows = (1 << 32) // bb + 4097
    w = torch.zeros(rows * bb, dtype=torch.uint8, device="cuda")
    tail = 41
    p = weights(8, tail, cols, 4)
    w[-tail * bb:] = torch.from_numpy(p).cuda()
    for tokens, xk in ((1, "bf16"), (16, "bf16")):
        x, x64 = activations(tokens, cols, xk, 5)
        y = torch.empty(tokens, rows, device="cuda")
        g.matvec(8, y, w, x)
        want, bound = ref.product(*ref.decode(oracle, 8, p, tail, cols), x64)
        assert ref.outside(y[:, -tail:].cpu().numpy(), want, bound, "f32") == 0
        assert bool((y[:, :-tail] == 0).all())
    ids = torch.tensor([rows - 1, rows - tail, 0, rows, -1], device="cuda")
    e = torch.empty(5, cols, device="cuda")
    g.get_rows(8, e, w, ids)
    dec = oracle.dequantize(8, p).reshape(tail, cols)
    got = e.cpu().numpy()
    assert same_bits(got[0], dec[-1]) and same_bits(got[1], dec[0]) and not got[2:].any()


@pytest.mark.parametrize("ty", [1, 2, 8, 12, 14])
@pytest.mark.parametrize("rows", [15, 16, 17, 31, 47, 48, 49])
@pytest.mark.parametrize("tokens", [2, 7, 16])
def test_matvec_rows_beside_a_tile(oracle, ty, rows, tokens):
    """Tiles that end with the matrix are moved back to end with it: no row twice, none behind the last."""
    run_matvec(oracle, ty, rows, 512, tokens, ("f32", "f16", "bf16")[rows % 3], "f32", rows + tokens, y_stride=rows + 5)


@pytest.mark.parametrize("ty,rows,cols,tokens,xk", [
    (12, 4097, 256, 2, "bf16"), (12, 8195, 2304, 16, "bf16"), (14, 12003, 512, 9, "f32"), (8, 30001, 256, 3, "f16"), (2, 4100, 4128, 16, "f32"),
    (30, 9001, 264, 5, "f16"), (1, 6005, 777, 8, "bf16"), (23, 5001, 2816, 16, "f16"), (10, 70001, 256, 2, "f32"), (15, 300, 16640, 16, "f32")])
def test_matvec_cuts(oracle, ty, rows, cols, tokens, xk):
    """From few to many rows and columns: one to three tiles a workgroup, one to eight waves that share its columns."""
    run_matvec(oracle, ty, rows, cols, tokens, xk, "f32", rows + cols)


@pytest.mark.parametrize("ty", [2, 12, 14, 20, 1, 30])
@pytest.mark.parametrize("tokens", [1, 3])
def test_matvec_subnormal_x(oracle, ty, tokens):
    """f16 x below 2^-14, whose every bit counts.  The products are far above the bounds of f32 sums."""
    import torch
    import gguf_amd as g
    rows, cols = 33, 512
    p = weights(ty, rows, cols, ty)
    v = np.random.default_rng(ty).integers(-1023, 1024, (tokens, cols)) * 2.0 ** -24
    x = torch.from_numpy(v).cuda().to(torch.float16)
    assert bool((x.double().cpu().numpy() == v).all())
    y = torch.empty(tokens, rows, device="cuda")
    g.matvec(ty, y, on_device(p), x)
    torch.cuda.synchronize()
    want, bound = ref.product(*ref.decode(oracle, ty, p, rows, cols), v)
    assert ref.outside(y.cpu().numpy(), want, bound, "f32") == 0


# ---- rows by id --------------------------------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("yk", ["f32", "f16", "bf16"])
def test_get_rows(oracle, ty, yk):
    """Bit for bit what the decode kernels write; ids twice, outside, and of both widths; rows at odd distances."""
    import torch
    import gguf_amd as g
    for rows, cols, n, wide, pad, offset in ((50, 768, 33, True, 0, 0), (7, 256, 1, False, 3, 2), (300, 2304, 100, False, 8, 1), (9, 1280, 5, True, 1, 4)):
        if ty in (1, 30):
            cols += 5
        p = weights(ty, rows, cols, ty + rows)
        ids = np.random.default_rng(n).integers(0, rows, n)
        ids[n // 2] = ids[0]
        if n > 3:
            ids[1], ids[2] = -1, rows
        buf, y = output(n, cols, yk, cols + pad)
        g.get_rows(ty, y, on_device(p, offset), torch.from_numpy(ids).to(torch.int64 if wide else torch.int32).cuda())
        torch.cuda.synchronize()
        dec = oracle.dequantize(ty, p, KIND[yk]).reshape(rows, cols)
        want = np.where(((ids >= 0) & (ids < rows))[:, None], dec[np.clip(ids, 0, rows - 1)], np.zeros((), dec.dtype))
        got = y.contiguous()
        if yk == "f32":
            assert same_bits(got.cpu().numpy(), want)
        else:
            assert same_bits16(got.view(torch.int16).cpu().numpy(), want, yk)
        assert untouched(buf, n, cols)


def test_get_rows_extreme_ids():
    import torch
    import gguf_amd as g
    w = torch.full((4 * 34,), 1, dtype=torch.uint8, device="cuda")
    ids = torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 32, 2 ** 32 + 1, 4, 3], device="cuda")
    y = torch.full((6, 32), 5.0, device="cuda")
    g.get_rows(8, y, w, ids)
    assert not y[:5].cpu().numpy().any() and y[5].cpu().numpy().all()
    z = torch.full((2, 32), 5.0, device="cuda")
    g.get_rows(8, z, w[:0], torch.zeros(2, dtype=torch.int32, device="cuda"))      # an empty table
    assert not z.cpu().numpy().any()


# ---- mixture of experts ------------------------------------------------------------------------------

class Moe:
    def __init__(self, oracle, experts, hidden, ff, ut, dt, router="f32", seed=0, **kw):
        import torch
        import gguf_amd as g
        rng = np.random.default_rng(seed)
        r = torch.from_numpy((rng.standard_normal((experts, hidden)) * 1.5 / hidden ** 0.5).astype(np.float32)).cuda().to(dtype(router))
        self.experts, self.hidden, self.ff = experts, hidden, ff
        self.kw = dict(top_k=2, gating="softmax", normalize=True, scale=1.0, activation="silu")
        self.kw.update(kw)
        self.router = r
        packs = [weights(ty, experts * a, b, seed + i) for i, (ty, a, b) in enumerate(((ut, ff, hidden), (ut, ff, hidden), (dt, hidden, ff)))]
        for ty, p in zip((ut, ut, dt), packs):                   # values near 0.02, as a model's
            be, bb = g.block_elems(ty), g.block_bytes(ty)
            if ty not in (1, 30):
                from gguf_amd import synth
                small = {2: 2 ** -8, 3: 2 ** -8, 6: 2 ** -9, 7: 2 ** -9, 8: 2 ** -12, 9: 2 ** -12, 10: 2 ** -9, 11: 2 ** -11, 12: 2 ** -13,
                         13: 2 ** -14, 14: 2 ** -15, 15: 2 ** -12, 20: 2 ** -12, 23: 2 ** -16}[ty]
                for off in synth.HEADER_F16[ty]:
                    p.reshape(-1, bb)[:, off:off + 2] = np.frombuffer(np.float16(small).tobytes(), dtype=np.uint8)
        def split(ty, p, rows, cols):
            return [ref.decode(oracle, ty, q, rows, cols) for q in p.reshape(experts, -1)]
        self.ref = [split(ut, packs[0], ff, hidden), split(ut, packs[1], ff, hidden), split(dt, packs[2], hidden, ff)]
        self.layer = g.MoeLayer(r, (ut, on_device(packs[0])), (ut, on_device(packs[1])), (dt, on_device(packs[2])), hidden=hidden, ff=ff, **self.kw)

    def check(self, x, yk, pad=0):
        import torch
        n = x.shape[0]
        buf, y = output(n, self.hidden, yk, self.hidden + pad)
        ids = torch.full((n, self.kw["top_k"]), -7, dtype=torch.int32, device="cuda")
        w = torch.empty(n, self.kw["top_k"], device="cuda")
        self.layer.run(y, x, ids=ids, weights=w)
        torch.cuda.synchronize()
        want, bound, wi, ww = ref.moe(self.router.double().cpu().numpy(), *self.ref, x.double().cpu().numpy(), **self.kw)
        assert np.array_equal(ids.cpu().numpy(), wi)
        assert np.allclose(w.cpu().numpy(), ww, rtol=(24 + self.experts) * ref.U * 16, atol=1e-30)
        got = y.float().cpu().numpy()
        assert ref.outside(got, want, bound, yk) == 0, np.abs(got - want).max()
        assert untouched(buf, n, self.hidden)


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 16])
@pytest.mark.parametrize("experts,top_k,hidden,ff,ut,dt,xk,yk,more", [
    (8, 2, 512, 768, 12, 14, "bf16", "bf16", {}),
    (4, 4, 256, 256, 2, 8, "f32", "f32", {"normalize": False}),
    (60, 8, 256, 512, 12, 13, "f16", "f32", {"gating": "sigmoid", "scale": 2.5}),
    (9, 3, 96, 160, 20, 3, "f32", "f16", {"activation": "gelu"}),
    (5, 1, 288, 64, 8, 2, "bf16", "f32", {"gating": "sigmoid", "normalize": False, "router": "bf16"}),
    (130, 5, 512, 256, 23, 10, "f32", "f32", {"router": "f16"}),
    (3, 2, 33, 47, 1, 30, "f32", "f32", {}),
    (6, 2, 1184, 2304, 6, 11, "bf16", "f32", {}),
    (2, 2, 256, 512, 15, 9, "f16", "f16", {}),
    (512, 32, 64, 32, 7, 20, "f32", "f32", {})])
def test_moe(oracle, tokens, experts, top_k, hidden, ff, ut, dt, xk, yk, more):
    m = Moe(oracle, experts, hidden, ff, ut, dt, seed=experts + tokens, top_k=top_k, **more)
    x, _ = activations(tokens, hidden, xk, tokens, hidden + 3)
    m.check(x, yk, pad=tokens % 3)


@pytest.mark.parametrize("ty", TYPES)
def test_moe_every_type(oracle, ty):
    hidden, ff = (512, 256) if ty not in (1, 30) else (77, 35)
    m = Moe(oracle, 7, hidden, ff, ty, ty, seed=ty, top_k=3)
    for tokens, xk in ((1, "bf16"), (6, "f32")):
        x, _ = activations(tokens, hidden, xk, tokens)
        m.check(x, "f32")


def test_moe_most_tokens_and_one_crowded_expert(oracle):
    m = Moe(oracle, 12, 256, 512, 12, 12, seed=4, top_k=2)
    x, _ = activations(64, 256, "f32", 9)
    m.check(x, "f32")
    same = x[:1].expand(64, 256)                                  # every token takes the same two experts
    m.check(same, "f32")
    m.check(x[:33], "bf16")


def test_moe_equal_logits_take_the_lowest_index(oracle):
    import torch
    m = Moe(oracle, 70, 256, 256, 2, 2, seed=4, top_k=6)
    m.router[:] = 0.0
    m.router[40] = m.router[7] = torch.randn(256, generator=torch.Generator().manual_seed(1)).cuda()
    x, _ = activations(4, 256, "f32", 9)
    m.check(x, "f32")
    y, ids = torch.empty(1, 256, device="cuda"), torch.empty(1, 6, dtype=torch.int32, device="cuda")
    m.layer.run(y, torch.zeros(1, 256, device="cuda"), ids=ids)
    assert ids.cpu().tolist() == [[0, 1, 2, 3, 4, 5]] and not y.cpu().numpy().any()


def test_moe_non_finite_token_stays_alone(oracle):
    """A NaN or an infinity in one token: its ids stay valid and different, the other tokens are what they were."""
    import torch
    m = Moe(oracle, 9, 512, 256, 12, 14, seed=2, top_k=3)
    x, _ = activations(5, 512, "f32", 1)
    x = x.clone()
    clean = torch.empty(5, 512, device="cuda")
    m.layer.run(clean, x)
    x[1, 3], x[3, 500] = float("nan"), float("inf")
    y, ids = torch.empty(5, 512, device="cuda"), torch.empty(5, 3, dtype=torch.int32, device="cuda")
    m.layer.run(y, x, ids=ids)
    torch.cuda.synchronize()
    got = ids.cpu().numpy()
    assert all(len(set(r)) == 3 and min(r) >= 0 and max(r) < 9 for r in got.tolist())
    y, clean = y.cpu().numpy(), clean.cpu().numpy()
    assert np.isnan(y[1]).all() and not np.isfinite(y[3]).any()
    want, bound, *_ = ref.moe(m.router.double().cpu().numpy(), *m.ref, x[[0, 2, 4]].double().cpu().numpy(), **m.kw)
    assert ref.outside(y[[0, 2, 4]], want, bound, "f32") == 0


@pytest.mark.parametrize("experts,top_k,tokens", [
    (2, 1, 6), (2, 2, 64), (2, 1, 33), (1, 1, 17), (7, 3, 9), (4, 1, 16), (4, 1, 17), (300, 4, 12), (64, 32, 4), (512, 2, 64), (65, 8, 8)])
def test_moe_tokens_of_an_expert(oracle, experts, top_k, tokens):
    """Experts with one token to all of them, some with more than a workgroup takes, and experts with none."""
    m = Moe(oracle, experts, 64, 96, 2, 8, seed=experts + tokens, top_k=top_k)
    for xk in ("f32", "bf16"):
        x, _ = activations(tokens, 64, xk, tokens)
        m.check(x, "f32", pad=1)


@pytest.mark.parametrize("tokens", [1, 3])
def test_moe_nan_logits_come_last(oracle, tokens):
    """Experts whose logit is NaN are chosen behind all others, the lowest index first."""
    import torch
    m = Moe(oracle, 6, 256, 256, 2, 2, seed=8, top_k=5)
    m.router[1] = m.router[2] = m.router[4] = float("nan")
    x, _ = activations(tokens, 256, "f32", 2)
    y, ids = torch.empty(tokens, 256, device="cuda"), torch.empty(tokens, 5, dtype=torch.int32, device="cuda")
    m.layer.run(y, x, ids=ids)
    got = ids.cpu().numpy()
    assert (np.sort(got[:, :3]) == [0, 3, 5]).all() and (got[:, 3:] == [1, 2]).all()
    logits = (x.double().cpu().numpy() @ np.nan_to_num(m.router.double().cpu().numpy()).T)
    assert all((np.diff(logits[t, got[t, :3]]) <= 0).all() for t in range(tokens))


def test_moe_same_result_alone_and_with_others(oracle):
    """A token's ids and weights do not depend on the tokens beside it."""
    import torch
    m = Moe(oracle, 20, 256, 256, 12, 12, seed=3, top_k=4)
    x, _ = activations(16, 256, "f32", 5)
    def run(x):
        n = x.shape[0]
        y, ids, w = torch.empty(n, 256, device="cuda"), torch.empty(n, 4, dtype=torch.int32, device="cuda"), torch.empty(n, 4, device="cuda")
        m.layer.run(y, x, ids=ids, weights=w)
        return ids, w
    ids, w = run(x)
    for n in (1, 2, 5):
        i, v = run(x[:n])
        assert torch.equal(i, ids[:n]) and same_bits(v.cpu().numpy(), w[:n].cpu().numpy())


def test_moe_graph_and_streams(oracle):
    """Replayed with new inputs (other experts), and two calls at once on two streams: each what it is alone."""
    import torch
    m = Moe(oracle, 16, 512, 768, 12, 14, seed=6, top_k=4)
    x, _ = activations(3, 512, "f32", 1)
    x = x.contiguous()
    y = torch.empty(3, 512, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.layer.run(y, x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.layer.run(y, x)
    for rep in range(4):
        x.copy_(torch.randn(3, 512, generator=torch.Generator().manual_seed(rep)))
        graph.replay()
        torch.cuda.synchronize()
        again = torch.empty_like(y)
        m.layer.run(again, x)
        torch.cuda.synchronize()
        assert torch.equal(again, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [activations(n, 512, "bf16", n)[0] for n in (1, 7)]
    outs = [[torch.empty(n, 512, device="cuda") for _ in range(6)] for n in (1, 7)]
    torch.cuda.synchronize()
    for k in range(6):
        for s, a, o in zip(streams, xs, outs):
            m.layer.run(o[k], a, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for a, o in zip(xs, outs):
        alone = torch.empty_like(o[0])
        m.layer.run(alone, a)
        torch.cuda.synchronize()
        assert all(torch.equal(v, alone) for v in o)


# ---- together ----------------------------------------------------------------------------------------

def test_a_decoding_step_through_packed_weights(oracle):
    """Embedding, a projection, a mixture-of-experts layer and the output head, one behind the other in one graph: each
    stage against 64 bits on the values that the stage before handed it."""
    import torch
    import gguf_amd as g
    hidden, vocab = 512, 1000
    emb, proj, head = weights(12, vocab, hidden, 1), weights(2, hidden, hidden, 2), weights(14, vocab, hidden, 3)
    demb, dproj, dhead = on_device(emb), on_device(proj), on_device(head)
    m = Moe(oracle, 8, hidden, 768, 12, 14, seed=8)
    for tokens in (1, 4):
        ids = torch.zeros(tokens, dtype=torch.int64, device="cuda")
        e, a, b = (torch.empty(tokens, hidden, device="cuda") for _ in range(3))
        logits = torch.empty(tokens, vocab, device="cuda")
        chosen = torch.empty(tokens, 2, dtype=torch.int32, device="cuda")

        def step():
            g.Q4K.get_rows(e, demb, ids)
            g.Q4_0.matvec(a, dproj, e)
            m.layer.run(b, a, ids=chosen)
            g.Q6K.matvec(logits, dhead, b)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for rep in range(3):
            ids.copy_(torch.randint(0, vocab, (tokens,), generator=torch.Generator().manual_seed(rep)))
            graph.replay()
            torch.cuda.synchronize()
            assert same_bits(e.cpu().numpy(), oracle.dequantize(12, emb).reshape(vocab, hidden)[ids.cpu().numpy()])
            for out, (ty, p, rows), src in ((a, (2, proj, hidden), e), (logits, (14, head, vocab), b)):
                want, bound = ref.product(*ref.decode(oracle, ty, p, rows, hidden), src.double().cpu().numpy())
                assert ref.outside(out.cpu().numpy(), want, bound, "f32") == 0
            want, bound, wi, _ = ref.moe(m.router.double().cpu().numpy(), *m.ref, a.double().cpu().numpy(), **m.kw)
            assert np.array_equal(chosen.cpu().numpy(), wi)
            assert ref.outside(b.cpu().numpy(), want, bound, "f32") == 0
