"""Products with packed weights on the GPU, at the ends of their ranges: rows that end a few elements into a turn, one token's
activations of every size, codes that are small beside their range, non-finite values, and long lists of ids."""
import numpy as np
import pytest

import matmul_ref as ref
from test_gpu_matmul import SENTINEL, Moe, activations, dtype, on_device, output, run_matvec, untouched, weights
from util import same_bits

pytestmark = pytest.mark.gpu


# ---- rows whose last turn is shorter than 16 bytes (tests/test_tile_reads.py follows the addresses on the CPU) ----------------

@pytest.mark.parametrize("ty", [1, 30])
@pytest.mark.parametrize("rows,cols,tokens", [(5, 1025, 1), (8, 1031, 1), (9, 2049, 1), (1, 1026, 1), (33, 3078, 1), (1, 257, 2), (1, 263, 16), (1, 513, 3),
                                              (17, 257, 2), (2, 2055, 7)])
def test_rows_that_end_a_few_elements_into_a_turn(oracle, ty, rows, cols, tokens):
    for xk in ("f32", "bf16"):
        run_matvec(oracle, ty, rows, cols, tokens, xk, "f32", rows + cols)


@pytest.mark.parametrize("ty", [1, 30])
@pytest.mark.parametrize("tokens", [1, 3])
def test_moe_rows_that_end_a_few_elements_into_a_turn(oracle, ty, tokens):
    for hidden, ff in ((257, 1), (259, 9), (1, 513), (9, 262)):
        m = Moe(oracle, 3, hidden, ff, ty, ty, seed=hidden + tokens)
        x, _ = activations(tokens, hidden, "f32", tokens)
        m.check(x, "f32", pad=1)


# ---- one token: what its activations are taken to ----------------------------------------------------------------------------

def one_token(ty, p, rows, cols, v, xk, yk):
    """(y, x in 64 bits) of packed rows p times the row of values v."""
    import torch
    import gguf_amd as g
    x = torch.from_numpy(np.asarray(v, dtype=np.float32)[None]).cuda().to(dtype(xk))
    y = torch.empty(1, rows, dtype=dtype(yk), device="cuda")
    g.matvec(ty, y, on_device(p), x)
    torch.cuda.synchronize()
    return y.float().cpu().numpy(), x.double().cpu().numpy()


def small_codes(ty, p):
    """Codes whose values are small beside the range that the type's codes have."""
    import gguf_amd as g
    b = p.reshape(-1, g.block_bytes(ty))
    if ty in (8, 9, 15):                              # within +-10
        lo = {8: 2, 9: 4, 15: 2}[ty]
        q = b[:, lo:lo + g.block_elems(ty)].astype(np.int16) % 21 - 10
        b[:, lo:lo + g.block_elems(ty)] = q.astype(np.int8).view(np.uint8)
    elif ty in (20, 23):                              # the code book's -10 and 1
        lo = {20: 2, 23: 8}[ty]
        b[:, lo:] = 0x77 + (b[:, lo:] & 0x11)
    else:                                             # q6_k: 32 to 39, values 0 to 7
        b[:, :128] &= 0x77
        b[:, 128:192] = 0xAA
    return p


@pytest.mark.parametrize("ty", [8, 9, 14, 15, 20, 23])
@pytest.mark.parametrize("xk,yk", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
def test_one_token_small_codes(oracle, ty, xk, yk):
    """The error goes by the weights' own size: no offset of the codes in the bound."""
    rows, cols = 777, 2048
    p = small_codes(ty, weights(ty, rows, cols, ty))
    got, x = one_token(ty, p, rows, cols, np.random.default_rng(ty).standard_normal(cols), xk, yk)
    w, _ = ref.decode(oracle, ty, p, rows, cols)
    want, bound = ref.product(w, np.zeros_like(w), x)
    assert ref.outside(got, want, bound, yk) == 0, np.abs(got - want).max()


@pytest.mark.parametrize("ty", [2, 8, 9, 15])
@pytest.mark.parametrize("xk,yk", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16")])
def test_one_token_beside_an_outlier(oracle, ty, xk, yk):
    """One of 32 neighbours is 2^10 times the others and meets a weight of 0: the others count in full.  Bound: the worst of the
    roundings of f32 sums, 16 for a sub-block and its scale, 2 for each sub-block in the row's sum, 24 to join the row's parts,
    of the sum of all magnitudes; and 2^-32 of the outlier for each element, half a step of 32 bits below 2^11."""
    import gguf_amd as g
    rows, cols = 300, 256
    p = weights(ty, rows, cols, ty + 5)
    b = p.reshape(-1, g.block_bytes(ty))
    if ty == 2:
        b[:, 2] = b[:, 2] & 0xF0 | 8
    else:
        b[:, {8: 2, 9: 4, 15: 2}[ty]::32][:, :g.block_elems(ty) // 32] = 0
    v = np.random.default_rng(ty).standard_normal(cols)
    v[::32] = 1024.0
    got, x = one_token(ty, p, rows, cols, v, xk, yk)
    w, w0 = ref.decode(oracle, ty, p, rows, cols)
    assert not w[:, ::32].any()
    bound = (40 + 2 * cols // 32) * ref.U * (np.abs(x) @ (np.abs(w - w0) + np.abs(w0)).T) + 2.0 ** -32 * 1024 * np.abs(w).sum(axis=1)
    assert ref.outside(got, x @ w.T, bound, yk) == 0, np.abs(got - x @ w.T).max()


@pytest.mark.parametrize("ty", [8, 9, 15])
def test_one_token_codes_of_zero(oracle, ty):
    """Weights that are all 0 under scales that are not: exactly 0."""
    import gguf_amd as g
    p = weights(ty, 40, 1024, ty)
    lo = {8: 2, 9: 4, 15: 2}[ty]
    p.reshape(-1, g.block_bytes(ty))[:, lo:lo + g.block_elems(ty)] = 0
    got, _ = one_token(ty, p, 40, 1024, np.random.default_rng(1).standard_normal(1024), "f32", "f32")
    assert not got.any()


@pytest.mark.parametrize("ty", [2, 3, 8, 10, 12, 14, 20, 23])
@pytest.mark.parametrize("xk,yk,low,high", [("f32", "f32", -118, 60), ("f32", "f32", -118, -112), ("bf16", "bf16", -125, -119), ("bf16", "f32", -125, 60),
                                            ("f16", "f16", -24, 10), ("f16", "f16", -24, -14), ("f32", "f32", 70, 98)])
def test_one_token_of_every_size(oracle, ty, xk, yk, low, high):
    """One block of 32 neighbours is small, the next large, and all of them may be small: down to where x's last bit is that of
    the smallest f32, up to where codes times x stay in range.  Weights below 4, results that y's type holds."""
    import gguf_amd as g
    from gguf_amd import synth
    rows, cols = 130, 1024
    p = weights(ty, rows, cols, ty)
    rng = np.random.default_rng(1000 + low + ty)
    b = p.reshape(-1, g.block_bytes(ty))
    for at in synth.HEADER_F16[ty]:
        d = (2.0 ** (-12 if g.block_elems(ty) == 256 else -6) * (1 + rng.random(len(b)))).astype(np.float16)
        b[:, at:at + 2] = d.view(np.uint8).reshape(-1, 2)
    v = rng.standard_normal(cols) * 2.0 ** (np.repeat(rng.integers(low + 3, high - 1, cols // 32), 32))
    got, x = one_token(ty, p, rows, cols, v, xk, yk)
    assert np.isfinite(x).all()
    want, bound = ref.product(*ref.decode(oracle, ty, p, rows, cols), x)
    assert ref.outside(got, want, bound, yk) == 0, np.abs(got - want).max()


@pytest.mark.parametrize("ty", [8, 9, 15])
def test_one_token_is_rounded_without_a_bias(oracle, ty):
    """Elements 2^-24 of the largest among 32 keep eight bits behind the point.  Rounded to nearest, x of one sign and weights of
    one sign are off by independent errors of at most half a step, 2^-8, which spread like 2^-8 / sqrt(3) sqrt(sum of w^2); six
    times that is never met.  Cut off, they would all have one sign: half a step for each of them, 4.6 times the bound."""
    import gguf_amd as g
    rows, cols = 200, 256
    p = weights(ty, rows, cols, ty)
    b = p.reshape(-1, g.block_bytes(ty))
    lo = {8: 2, 9: 4, 15: 2}[ty]
    b[:, lo:lo + g.block_elems(ty)] = 10
    b[:, lo:lo + g.block_elems(ty):32] = 0
    v = 1.0 + np.random.default_rng(ty).random(cols)
    v[::32] = 2.0 ** 24
    got, x = one_token(ty, p, rows, cols, v, "f32", "f32")
    w, _ = ref.decode(oracle, ty, p, rows, cols)
    bound = 6 * 2.0 ** -8 / 3 ** 0.5 * np.sqrt((w ** 2).sum(axis=1)) + (40 + 2 * cols // 32) * ref.U * (x @ w.T)
    assert ref.outside(got, x @ w.T, bound, "f32") == 0, (np.abs(got - x @ w.T) / bound).max()


PACKED = [2, 3, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 20, 23]


@pytest.mark.parametrize("ty", PACKED + [1, 30])
@pytest.mark.parametrize("xk,yk", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
def test_one_token_non_finite_x(oracle, ty, xk, yk, bad):
    """Wherever it stands, in the first sub-block or another, in the first chunk of x or a later one."""
    rows, cols = 37, 1536
    p = weights(ty, rows, cols, ty)
    for at in (0, 31, 700, 1535):
        v = np.random.default_rng(at).standard_normal(cols)
        v[at] = float(bad)
        got, _ = one_token(ty, p, rows, cols, v, xk, yk)
        assert not np.isfinite(got).any(), at


@pytest.mark.parametrize("ty", PACKED + [1, 30])
@pytest.mark.parametrize("tokens", [1, 2])
def test_non_finite_scale_stays_in_its_row(oracle, ty, tokens):
    import torch
    import gguf_amd as g
    from gguf_amd import synth
    rows, cols, row = 37, 1536, 21
    bb, be = g.block_bytes(ty), g.block_elems(ty)
    for bits in (0x7C00, 0xFC00, 0x7E00) if ty != 30 else (0x7F80, 0xFF80, 0x7FC0):
        p = weights(ty, rows, cols, ty)
        at = row * (cols // be) * bb + 2 * bb + (synth.HEADER_F16[ty][0] if ty in PACKED else 0)
        p[at:at + 2] = np.frombuffer(np.uint16(bits).tobytes(), dtype=np.uint8)
        x, x64 = activations(tokens, cols, "f32", 3)
        buf, y = output(tokens, rows, "f32", rows + 3)
        g.matvec(ty, y, on_device(p), x)
        torch.cuda.synchronize()
        p[at:at + 2] = 0
        want, bound = ref.product(*ref.decode(oracle, ty, p, rows, cols), x64)
        got, others = y.cpu().numpy(), [r for r in range(rows) if r != row]
        assert ref.outside(got[:, others], want[:, others], bound[:, others], "f32") == 0
        assert not np.isfinite(got[:, row]).any()
        assert untouched(buf, tokens, rows)


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("ut,dt,xk", [(12, 14, "f32"), (2, 8, "bf16"), (20, 23, "f16"), (1, 30, "f32")])
def test_moe_one_token_non_finite(oracle, bad, ut, dt, xk):
    """The ids stay valid and different; the layer's next call is what it was."""
    import torch
    m = Moe(oracle, 9, 512, 256, ut, dt, seed=2, top_k=3)
    x, _ = activations(1, 512, xk, 1)
    hurt = x.clone()
    hurt[0, 300] = float(bad)
    y, ids = torch.empty(1, 512, device="cuda"), torch.full((1, 3), -7, dtype=torch.int32, device="cuda")
    m.layer.run(y, hurt, ids=ids)
    torch.cuda.synchronize()
    got = ids.cpu().numpy()[0].tolist()
    assert len(set(got)) == 3 and min(got) >= 0 and max(got) < 9
    assert not np.isfinite(y.cpu().numpy()).any()
    m.check(x, "f32")


# ---- several tokens ------------------------------------------------------------------------------------------------------------

def test_moe_keeps_32_bits_between_its_products():
    """Whole numbers in, so that gate and up are exact in any order, and a `down` that picks one element for each output: 16-bit
    outputs are the f32 outputs rounded once."""
    import torch
    import gguf_amd as g
    n = 256
    rng = np.random.default_rng(3)

    def q8_0(codes, d):
        b = np.zeros((codes.size // 32, 34), dtype=np.uint8)
        b[:, :2] = np.frombuffer(np.float16(d).tobytes(), dtype=np.uint8)
        b[:, 2:] = codes.astype(np.int8).view(np.uint8).reshape(-1, 32)
        return on_device(b.reshape(-1))

    gate, up = (q8_0(rng.integers(-3, 4, (2, n, n)), d) for d in (2.0 ** -6, 2.0 ** -3))
    down = q8_0(np.stack([np.eye(n), np.eye(n)]), 1.0)
    layer = g.MoeLayer(torch.randn(2, n, device="cuda"), (8, gate), (8, up), (8, down), hidden=n, ff=n, top_k=1)
    for xk in ("f16", "bf16"):
        x = torch.from_numpy(rng.integers(-8, 9, (16, n)).astype(np.float32)).cuda().to(dtype(xk))
        wide, y = torch.empty(16, n, device="cuda"), torch.empty(16, n, dtype=dtype(xk), device="cuda")
        layer.run(wide, x)
        layer.run(y, x)
        torch.cuda.synchronize()
        assert wide.unique().numel() > 2000
        assert torch.equal(y, wide.to(dtype(xk)))


@pytest.mark.parametrize("ty", [1, 2, 12, 14, 30])
@pytest.mark.parametrize("tokens", [2, 9])
def test_several_tokens_of_every_size(oracle, ty, tokens):
    """As for one token; of f32 x the bits below 2^-133 are left out."""
    import torch
    import gguf_amd as g
    rows, cols = 70, 1024
    p = weights(ty, rows, cols, ty)
    for xk, low, high in (("f32", -118, 60), ("f32", -118, -112), ("f32", -126, -120), ("bf16", -125, -119), ("f16", -24, -14), ("f32", 70, 98)):
        rng = np.random.default_rng(1000 + low + ty)
        v = rng.standard_normal((tokens, cols)) * 2.0 ** np.repeat(rng.integers(low + 3, high - 1, (tokens, cols // 32)), 32, axis=1)
        x = torch.from_numpy(v.astype(np.float32)).cuda().to(dtype(xk))
        y = torch.empty(tokens, rows, device="cuda")
        g.matvec(ty, y, on_device(p), x)
        torch.cuda.synchronize()
        w, w0 = ref.decode(oracle, ty, p, rows, cols)
        want, bound = ref.product(w, w0, x.double().cpu().numpy())
        # what is left out of an element meets its weight; a sub-block's offset meets the same sum of x
        floor = 2.0 ** -133 * (np.abs(w)).sum(axis=1) if xk == "f32" else 0.0
        assert ref.outside(y.cpu().numpy(), want, bound + floor, "f32") == 0, (xk, low)


@pytest.mark.parametrize("ty", [1, 8, 14])
@pytest.mark.parametrize("tokens", [1, 2])
def test_rows_near_the_longest(ty, tokens):
    """Rows of nearly 2^26 elements, sixteen to a tile: nearly 2^31 bytes of 16-bit floats.  Whole numbers at a few places of each
    row, zeros elsewhere: every sum is exact."""
    import torch
    import gguf_amd as g
    be, bb = g.block_elems(ty), g.block_bytes(ty)
    rows, cols = 17, (1 << 26) - (5 if ty == 1 else be)
    w = torch.zeros(rows * (cols // be), bb, dtype=torch.uint8, device="cuda")
    one = np.frombuffer(np.float16(1.0).tobytes(), dtype=np.uint8)
    # block 0 of every type here: one code of the first element's is 1, its scale is 1
    block = np.zeros(bb, dtype=np.uint8)
    if ty == 1:
        block[:] = one
    elif ty == 8:
        block[:2], block[2] = one, 1
    else:                                              # q6_k: 32 is 0, 33 is 1; all scales are 1
        block[128:192], block[192:208], block[208:], block[0] = 0xAA, 1, one, 1
    blocks = cols // be
    places = [0, blocks // 3, blocks - 1]
    for r in range(rows):
        for b in places[:1 + r % 3]:
            w[r * blocks + b] = torch.from_numpy(block).cuda()
    x = torch.zeros(tokens, cols, device="cuda")
    for t in range(tokens):
        for i, b in enumerate(places):
            x[t, b * be] = 10.0 ** i * (t + 1)
    y = torch.empty(tokens, rows, device="cuda")
    g.matvec(ty, y, w.view(-1), x)
    want = [[(t + 1) * float("111"[: 1 + r % 3]) for r in range(rows)] for t in range(tokens)]
    assert y.cpu().tolist() == want


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("tokens", [1, 3])
def test_moe_activation_over_its_range(activation, tokens):
    """Gate values from -24 to 24 in steps of 1/16 and more, exact in any order, by an `up` of ones and a `down` that picks one element: the
    activation itself, in its own size.  32-bit roundings, half a unit each: z takes 5, each of which exp turns into 2 |z| of its
    result (SiLU: |z|, and none), exp, the sum, the quotient and two products below 8."""
    import torch
    import gguf_amd as g
    n = 512

    def q8_0(codes, d):
        b = np.zeros((codes.size // 32, 34), dtype=np.uint8)
        b[:, :2] = np.frombuffer(np.float16(d).tobytes(), dtype=np.uint8)
        b[:, 2:] = codes.astype(np.int8).view(np.uint8).reshape(-1, 32)
        return on_device(b.reshape(-1))

    # x = (t + 1, 1, 0, ..): gate = (t + 1) code 2^-4 in column 0, up = 1 in column 1
    codes = np.zeros((1, n, n))
    codes[0, :, 0] = np.arange(n) % 256 - 128
    ones = np.zeros((1, n, n))
    ones[0, :, 1] = 1
    layer = g.MoeLayer(torch.ones(1, n, device="cuda"), (8, q8_0(codes, 2.0 ** -4)), (8, q8_0(ones, 1.0)), (8, q8_0(np.eye(n)[None], 1.0)), hidden=n, ff=n,
                       top_k=1, activation=activation)
    x = torch.zeros(tokens, n, device="cuda")
    x[:, 0] = torch.arange(1, tokens + 1) if tokens > 1 else 2.0
    x[:, 1] = 1.0
    y = torch.empty(tokens, n, device="cuda")
    layer.run(y, x)
    torch.cuda.synchronize()
    v = (x[:, :1].double().cpu().numpy()) * codes[0, :, 0][None] * 2.0 ** -4
    z = v if activation == "silu" else 2.0 * np.sqrt(2.0 / np.pi) * (v + 0.044715 * v ** 3)
    with np.errstate(over="ignore"):
        want = v / (1.0 + np.exp(-z))
    tol = (8 + 10 * np.abs(z)) * ref.U * np.abs(want) + 2.0 ** -126
    if tokens == 1:
        # an element of h is taken to 2^-32 of the largest of 32 neighbours
        tol = tol + 2.0 ** -32 * np.repeat(np.abs(want).reshape(tokens, -1, 32).max(axis=2), 32, axis=1)
    assert (np.abs(y.cpu().numpy() - want) <= tol).all(), np.abs(y.cpu().numpy() - want).max()


def test_moe_workspace_belongs_to_the_stream_of_the_call(oracle, monkeypatch):
    """... also where that is the default stream, whose handle is 0: memory of another stream could be handed out again while
    the kernels still use it."""
    import torch
    m = Moe(oracle, 4, 256, 256, 2, 2, seed=1)
    x, _ = activations(2, 256, "f32", 1)
    y = torch.empty(2, 256, device="cuda")
    side = torch.cuda.Stream()
    owners, empty = [], torch.empty

    def spy(*args, **kw):
        owners.append(torch.cuda.current_stream().cuda_stream)
        return empty(*args, **kw)

    torch.cuda.synchronize()
    monkeypatch.setattr(torch, "empty", spy)
    for current in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(current):
            for stream in (None, 0, torch.cuda.default_stream().cuda_stream, side.cuda_stream):
                owners.clear()
                m.layer.run(y, x, stream=stream)
                torch.cuda.synchronize()
                assert owners == [current.cuda_stream if stream is None else stream]


@pytest.mark.parametrize("experts,top_k", [(512, 32), (40, 32)])
def test_moe_most_pairs(oracle, experts, top_k):
    """64 tokens of 32 experts each."""
    m = Moe(oracle, experts, 64, 32, 7, 20, seed=experts, top_k=top_k)
    x, _ = activations(64, 64, "f32", 5)
    m.check(x, "f32", pad=3)


@pytest.mark.parametrize("ty", [1, 2, 12, 14])
@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("xk", ["f32", "f16", "bf16"])
def test_x_and_y_begin_anywhere(oracle, ty, tokens, xk):
    """x and y at any multiple of their element size."""
    import torch
    import gguf_amd as g
    rows, cols = 37, 768
    p = weights(ty, rows, cols, ty)
    w, w0 = ref.decode(oracle, ty, p, rows, cols)
    m = Moe(oracle, 5, 256, 256, 2, ty if ty != 1 else 12, seed=ty)
    for off in (1, 3, 6):
        v, x64 = activations(1, tokens * cols + off, xk, off)
        x = v[0, off:].view(tokens, cols)
        out = torch.full((tokens * rows + off + 1,), SENTINEL, dtype=dtype(xk), device="cuda")
        y = out[off:-1].view(tokens, rows)
        g.matvec(ty, y, on_device(p), x)
        torch.cuda.synchronize()
        want, bound = ref.product(w, w0, x64[0, off:].reshape(tokens, cols))
        assert ref.outside(y.float().cpu().numpy(), want, bound, xk) == 0
        assert bool((out[:off] == SENTINEL).all()) and float(out[-1]) == SENTINEL
        m.check(v[0, off:off + tokens * 256].view(tokens, 256), xk)


# ---- rows by id ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("ty,cols", [(2, 32), (14, 256), (1, 5)])
def test_get_rows_of_more_ids_than_one_launch_takes(oracle, ty, cols):
    import torch
    import gguf_amd as g
    rows, n = 50, 2 * 65535 + 37
    p = weights(ty, rows, cols, ty)
    ids = np.random.default_rng(ty).integers(-1, rows + 1, n)
    buf, y = output(n, cols, "f32", cols + 1)
    g.get_rows(ty, y, on_device(p), torch.from_numpy(ids).cuda())
    torch.cuda.synchronize()
    dec = oracle.dequantize(ty, p).reshape(rows, cols)
    want = np.where(((ids >= 0) & (ids < rows))[:, None], dec[np.clip(ids, 0, rows - 1)], np.float32(0))
    assert same_bits(y.contiguous().cpu().numpy(), want)
    assert untouched(buf, n, cols)
