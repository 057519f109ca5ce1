"""The microscaled (MX) operators at sizes and shapes where launches, tiles and strides change."""
import pytest
import torch

from ditserve_amd import _lib, mx, ops
from tests.helpers import mx_gemm_plan

pytestmark = pytest.mark.gpu
DEV = "cuda"


def raw(m):
    return m.data.view(torch.uint8), m.scales.view(torch.uint8)


@pytest.mark.parametrize("op,cols", [("quantize", 32), ("quantize", 544), ("norm", 32)])
def test_more_rows_than_one_launch_dimension_holds(op, cols):
    """From 2^26 waves on a launch has 2^32 threads, which its first dimension does not hold: every row is
    written all the same.  Rows repeat with a period, so each is compared with its own of a small call."""
    rows, period = (1 << 26) // ((cols + 511) // 512 if op == "quantize" else 1) + 5, 4093
    g = torch.Generator(device=DEV).manual_seed(cols)
    few = torch.randn((period, cols), generator=g, device=DEV).to(torch.bfloat16)
    call = mx.quantize if op == "quantize" else mx.norm
    want = raw(call(few))
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=DEV)
    whole = rows // period * period
    x[:whole].view(-1, period, cols).copy_(few)
    x[whole:].copy_(few[:rows - whole])
    out = mx.MXTensor.empty(rows, cols, DEV)
    for t in raw(out):
        t.fill_(0xAA)
    call(x, out=out)
    for got, ref in zip(raw(out), want):
        parts = got[:whole].view(-1, period, got.shape[1])
        for i in range(0, parts.shape[0], 1024):
            assert (parts[i:i + 1024] == ref).all(), i
        assert torch.equal(got[whole:], ref[:rows - whole])


# ---------------------------------------------------------------------------------------------
# linear: the kernels by shape and stride, each asserted
# ---------------------------------------------------------------------------------------------

def decode(m):
    """(values over the scales, scales of each value) of an fp8 MX matrix in 64 bits, from its bytes, on the GPU."""
    data, scales = (t.long() for t in raw(m))
    e, f, sign = data >> 3 & 15, (data & 7).double() / 8, 1 - 2 * (data >> 7).double()
    v = sign * torch.where(e > 0, (1 + f) * torch.exp2((e - 7).double()), f * 2.0 ** -6)
    place = [16 * (i // 16) + 4 * (i % 4) + (i % 16) // 4 for i in range(m.cols // 32)]  # block i's byte
    return v[:, :m.cols], torch.exp2((scales[:, place] - 127).double()).repeat_interleave(32, 1)


def operand(rows, cols, seed, sub=0, pad=0):
    """MX rows of random values (scales lowered by 2^sub); pad: bytes behind each row of both tensors."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((rows, cols), generator=g, device=DEV) * torch.exp(torch.randn((rows, 1), generator=g, device=DEV))
    q = mx.quantize(x.to(torch.bfloat16))
    raw(q)[1].sub_(sub)
    return q if not pad else in_rows(q, q.data.shape[1] + pad, q.scales.shape[1] + pad)


def in_rows(q, data_stride, scale_stride):
    """The same matrix with row strides of its own."""
    parts = []
    for t, stride in zip(raw(q), (data_stride, scale_stride)):
        view = torch.empty(t.shape[0] * stride, dtype=torch.uint8, device=DEV).as_strided(t.shape, (stride, 1))
        parts.append(view.copy_(t))
    return mx.MXTensor("fp8", parts[0].view(torch.float8_e4m3fn), parts[1].view(torch.float8_e8m0fnu), q.cols)


def gated(M, N, seed):
    """Residual, gate and segments: an empty one, and ends inside tiles."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cu = [0, 1, 1, M // 3, M]
    return dict(epilogue="gate_res", residual=torch.randn((M, N), generator=g, device=DEV).to(torch.bfloat16),
                gate=torch.randn((4, N), generator=g, device=DEV), segments=ops.Segments(cu, DEV))


def same(a, b):
    if isinstance(a, mx.MXTensor):
        return all(torch.equal(x, y) for x, y in zip(raw(a), raw(b)))
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


WIDE = (1 << 23) + 16  # 256 rows of it pass 2^31 bytes


@pytest.mark.parametrize("mx_out", [False, True])
@pytest.mark.parametrize("M,N,K,wide,kernel", [(333, 1568, 1056, "x", 5), (1560, 320, 2464, "x", 5), (1300, 1568, 608, "w", 5),
                                               (4200, 2016, 1056, "w", 4), (4353, 2016, 672, "w", 4)])
def test_linear_wide_strides_of_long_k(M, N, K, wide, kernel, mx_out):
    """More than four stages of 128 k (both scale buffers) in the kernels with 64-bit addresses, bitwise the packed
    product's results, which other kernels compute."""
    x, w = operand(M, K, M + K), operand(N, K, N + K, 4)
    b = torch.randn(N, generator=torch.Generator(device=DEV).manual_seed(M), device=DEV)
    kw = dict(epilogue="gelu", out_fmt="fp8") if mx_out else gated(M, N, K)
    assert mx_gemm_plan(M, N, K, WIDE, mx_out) == (kernel, M, 0) and mx_gemm_plan(M, N, K, mx_out=mx_out)[0] not in (4, 5)
    want = mx.linear(x, w, b, **kw)
    wx, ww = (in_rows(q, WIDE, q.scales.shape[1] + 32) if name == wide else q for q, name in ((x, "x"), (w, "w")))
    assert same(mx.linear(wx, ww, b, **kw), want)


@pytest.mark.parametrize("M,N,K,plan", [
    (9000, 120, 1536, (3, 9000, 0)), (5000, 120, 448, (3, 5000, 0)), (5000, 96, 448, (3, 5000, 0)),
    (20000, 64, 1536, (2, 20000, 0)), (20000, 8, 2432, (2, 20000, 0)), (20000, 96, 672, (2, 20000, 0)),
    (40000, 200, 1536, (0, 40000, 0)), (70000, 200, 416, (0, 65536, 3)), (33000, 160, 160, (0, 33000, 0)),
    (25000, 200, 416, (1, 25000, 0)), (18000, 224, 672, (1, 18000, 0))])
def test_linear_tiles_wider_than_the_matrix(M, N, K, plan):
    """Tiles of the one-wave-per-SIMD kernel that reach past N: weight rows, scales, bias and gate behind the last
    feature are not read, outputs behind it not written.  Against 64 bits, and bitwise against a few of the
    rows alone, which single waves compute."""
    assert mx_gemm_plan(M, N, K) == plan
    x, w = operand(M, K, M + K, pad=64), operand(N, K, N + K, 4, pad=32)
    b = torch.randn(N, generator=torch.Generator(device=DEV).manual_seed(M), device=DEV)
    kw = gated(M, N, K)
    buf = torch.full((M + 2, N + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    out = mx.linear(x, w, b, out=buf[:M, 8:8 + N], **kw)
    assert (buf[M:] == 7).all() and (buf[:, :8] == 7).all() and (buf[:, 8 + N:] == 7).all()
    (xv, xs), (wv, ws) = decode(x), decode(w)
    y = torch.mm(xv * xs, (wv * ws).T) + b.double()
    # Of the products of 8 consecutive k the instruction keeps 13 bits below the largest sum of two factors' exponents, a
    # subnormal factor's being that of 2^-6: 8 * 2^-13 of it a group, taken as the sum of all; and 17 additions
    # with 24 bits for each 128 k.
    least = [torch.where(v == 0, 0.0, v.abs().clamp_min(2.0 ** -6)) * s for v, s in ((xv, xs), (wv, ws))]
    acc = (8 * 2.0 ** -13 + (K + 127) // 128 * 17 * 2.0 ** -23) * torch.mm(least[0], least[1].T)
    seg = torch.bucketize(torch.arange(M, device=DEV), torch.tensor(kw["segments"].cu[1:], device=DEV), right=True)
    gate = kw["gate"].double()[seg]
    want = kw["residual"].double() + y * gate
    err = (out.double() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + gate.abs() * (acc + 2.0 ** -22 * y.abs())).all()
    # in norm, where errors do not add up: uniform roundings to bf16, and 2^-15 of the magnitudes (1.6e-5 on random data)
    mag = torch.mm((xv * xs).abs(), (wv * ws).abs().T)
    assert (out.double() - want).norm() <= 2.0 ** -8 / 3 ** 0.5 * want.norm() + 2.0 ** -15 * (gate * mag).norm()
    rows = [0, 1, M // 3 - 1, M // 3, M // 2, M - 17]
    few = {i: mx.linear(x[i:i + 1], w, b) for i in rows}
    all_ = mx.linear(x, w, b)
    for i in rows:
        assert mx_gemm_plan(1, N, K)[0] in (6, 7) and same(all_[i:i + 1], few[i])
    if N % 32 == 0:
        whole = mx.MXTensor.empty(M + 2, N, DEV)
        for t in raw(whole):
            t.fill_(0xAA)
        got = mx.linear(x, w, b, epilogue="silu", out_fmt="fp8", out=whole[:M])
        assert all((t[M:] == 0xAA).all() for t in raw(whole))
        data, scales = raw(got)
        assert (data[:, N:] == 0).all()
        pad = [i for i in range(scales.shape[1]) if 16 * (i // 16) + 4 * (i % 4) + (i % 16) // 4 >= N // 32]
        assert (scales[:, pad] == 127).all()
        v, s = decode(got)
        z = y * torch.sigmoid(y)
        off = 1.13 * (acc + 2.0 ** -20 * y.abs())  # SiLU's slope is up to 1.1
        assert ((v * s - z).abs() <= 2.0 ** -4 * z.abs() + s * 2.0 ** -10 + 1.25 * off).all()
        for i in rows:
            assert same(got[i:i + 1], mx.linear(x[i:i + 1], w, b, epilogue="silu", out_fmt="fp8"))


def test_outputs_beside_their_operands():
    """Operands and outputs that are column ranges of one buffer."""
    g = torch.Generator(device=DEV).manual_seed(5)
    M, N = 333, 512
    wide = torch.randn((M + 1, 6 * N), generator=g, device=DEV).to(torch.bfloat16)
    part = [wide[:M, i * N:(i + 1) * N] for i in range(6)]
    kept = [p.clone() for p in part]
    want, h = mx.norm(kept[0], kept[1])
    got, h2 = mx.norm(part[0], part[1], residual_out=part[2])
    assert same(got, want) and torch.equal(part[2], h) and h2 is part[2]
    w, w4 = operand(N, N, 6), mx.quantize(kept[0].repeat(2, 1)[:N], "fp4")
    mx.linear(got, w, epilogue="res", residual=part[1], out=wide[1:, 3 * N:4 * N])
    assert torch.equal(wide[1:, 3 * N:4 * N], mx.linear(got, w, epilogue="res", residual=kept[1]))
    mx.matvec(part[0][:40], w4, epilogue="res", residual=part[1][:40], out=wide[:40, 4 * N:5 * N])
    assert torch.equal(wide[:40, 4 * N:5 * N], mx.matvec(kept[0][:40], w4, epilogue="res", residual=kept[1][:40]))
    assert all(torch.equal(part[i], kept[i]) for i in (0, 1, 5))


def mx_rows_in(rows, cols, extra=2):
    """An MX output inside wider rows, every byte of the buffers 0xAA."""
    d, s = (cols + 127) // 128 * 128, (cols + 511) // 512 * 16
    bufs = [torch.full((rows + extra, n + 48), 0xAA, dtype=torch.uint8, device=DEV) for n in (d, s)]
    views = [b[:rows, 16:16 + n] for b, n in zip(bufs, (d, s))]
    return bufs, mx.MXTensor("fp8", views[0].view(torch.float8_e4m3fn), views[1].view(torch.float8_e8m0fnu), cols)


def untouched(bufs, rows):
    return all((b[rows:] == 0xAA).all() and (b[:rows, :16] == 0xAA).all() and (b[:rows, -32:] == 0xAA).all() for b in bufs)


# every kernel (few rows, the tiles, the two with 64-bit addresses, a split launch)
KERNELS = [((16, 1536, 1536), (6, 16, 0)), ((100, 1568, 416), (7, 100, 0)), ((333, 4640, 1536), (3, 333, 0)),
           ((520, 4640, 448), (2, 520, 0)), ((700, 7328, 1056), (1, 700, 0)), ((1560, 8960, 512), (0, 1560, 0)),
           ((4353, 4128, 448), (0, 3840, 2)), ((2600, 8960, 512), (0, 1792, 1)), ((700, 4128, 288), (5, 700, 0)),
           ((2601, 4128, 96), (4, 2601, 0))]


@pytest.mark.parametrize("shape,plan", KERNELS)
def test_mx_outputs_in_wider_rows(shape, plan):
    M, N, K = shape
    assert mx_gemm_plan(*shape, mx_out=True) == plan
    x, w = operand(M, K, 1), operand(N, K, 2, 4, pad=16)
    bufs, out = mx_rows_in(M, N)
    assert same(mx.linear(x, w, epilogue="gelu", out_fmt="fp8", out=out), mx.linear(x, w, epilogue="gelu", out_fmt="fp8"))
    assert untouched(bufs, M)


@pytest.mark.parametrize("rows,cols", [(5, 96), (67, 2432), (300, 6144)])
def test_row_operators_in_wider_rows(rows, cols):
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, r = (torch.randn((rows, cols), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    bufs, out = mx_rows_in(rows, cols)
    assert same(mx.quantize(x, out=out), mx.quantize(x)) and untouched(bufs, rows)
    want, h = mx.norm(x, r)
    bufs, out = mx_rows_in(rows, cols)
    wide = torch.full((rows + 2, cols + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    got, h2 = mx.norm(x, r, out=out, residual_out=wide[:rows, 8:8 + cols])
    assert same(got, want) and torch.equal(h2, h) and untouched(bufs, rows)
    assert (wide[rows:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 8 + cols:] == 7).all()


@pytest.mark.parametrize("shape,plan", KERNELS)
def test_non_finite_values_stay_in_their_row_and_feature(shape, plan):
    """An operand block of NaN makes its row or feature NaN and no other; a NaN or infinity of the residual, bias or
    gate its own outputs; in an MX output the block of 32."""
    M, N, K = shape
    assert mx_gemm_plan(*shape) == mx_gemm_plan(*shape, mx_out=True) == plan
    x, w = operand(M, K, 1), operand(N, K, 2, 4)
    kw = gated(M, N, 3)
    b = torch.randn(N, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    clean, clean_mx = mx.linear(x, w, b, **kw), mx.linear(x, w, b, out_fmt="fp8")
    row, feature, last = M // 2, N // 3, K // 32 - 1
    byte = last // 16 * 16 + last % 4 * 4 + last % 16 // 4
    raw(x)[1][row, byte] = 255
    raw(w)[1][feature, byte] = 255
    b[N - 1] = float("inf")
    kw["residual"][M - 1, 5] = float("nan")
    kw["gate"][3, 9] = float("nan")
    hit = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    hit[row] = hit[:, feature] = hit[:, N - 1] = True
    own = hit.clone()
    own[M - 1, 5] = own[M // 3:, 9] = True
    got = mx.linear(x, w, b, **kw)
    assert torch.equal(~got.isfinite(), own) and torch.equal(got[~own], clean[~own])
    data, scales = raw(mx.linear(x, w, b, out_fmt="fp8"))
    blocks = hit.view(M, N // 32, 32).any(2)
    place = [16 * (i // 16) + 4 * (i % 4) + (i % 16) // 4 for i in range(N // 32)]
    assert torch.equal(scales[:, place] == 255, blocks)
    keep = ~blocks.repeat_interleave(32, 1)
    assert torch.equal(data[:, :N][keep], raw(clean_mx)[0][:, :N][keep])


@pytest.mark.parametrize("shape,plan", KERNELS)
def test_gate_of_one_segment_and_of_each_row(shape, plan):
    """One segment for all rows, and segments of one row: the tiles' gate by LDS and by row."""
    M, N, K = shape
    x, w = operand(M, K, 1), operand(N, K, 2, 4)
    g = torch.Generator(device=DEV).manual_seed(5)
    r = torch.randn((M, N), generator=g, device=DEV).to(torch.bfloat16)
    gate = torch.randn((1, N), generator=g, device=DEV)
    one = mx.linear(x, w, epilogue="gate_res", residual=r, gate=gate, segments=ops.Segments([0, M], DEV))
    each = mx.linear(x, w, epilogue="gate_res", residual=r, gate=gate.expand(M, N), segments=ops.Segments(range(M + 1), DEV))
    assert same(one, each)
    # and the ungated one under a gate of 1
    ones = mx.linear(x, w, epilogue="gate_res", residual=r, gate=torch.ones_like(gate), segments=ops.Segments([0, M], DEV))
    assert same(ones, mx.linear(x, w, epilogue="res", residual=r))


@pytest.mark.parametrize("shape,plan", [((300, 4640, 1536), (3, 300, 0)), ((1560, 8960, 512), (0, 1560, 0)),
                                        ((100, 1568, 416), (7, 100, 0)), ((700, 4128, 288), (5, 700, 0))])
def test_widest_output_and_residual_rows(shape, plan):
    """Rows of 2^22 - 8 elements, the longest that a tile's 32-bit offsets are used with, are written and read where
    they are; longer ones are refused."""
    M, N, K = shape
    assert mx_gemm_plan(*shape) == plan
    x, w, kw = operand(M, K, 1), operand(N, K, 2, 4), gated(M, N, 3)
    want = mx.linear(x, w, **kw)
    stride = (1 << 22) - 8
    flat = torch.empty(M * stride, dtype=torch.bfloat16, device=DEV)
    res = flat.as_strided((M, N), (stride, 1)).copy_(kw["residual"])
    out = flat.as_strided((M, N), (stride, 1), N).fill_(7.0)
    behind = flat.as_strided((M, 64), (stride, 1), 2 * N).fill_(7.0)
    assert mx.linear(x, w, **{**kw, "residual": res}, out=out) is out
    assert same(out, want) and torch.equal(res, kw["residual"]) and (behind == 7).all()
    over = flat.as_strided((M - 1, N), (stride + 8, 1))
    with pytest.raises(_lib.DitkError, match="strides too large"):
        mx.linear(x[:M - 1], w, out=over)
