"""The 4-bit layer (QLinear4) on the device against numpy in 64 bits: codes and scales bit for bit, forwards within
a bound that counts the kernel's roundings.

Forward bound, per element.  An activation is rounded to its group's grid, whose step is at most 2^-22 of the group's
largest |x|: off by 2^-23 of that, times sum|q| * scale.  Products and sums within a group are exact integers.  In units
of S = sum_i |x_i * q_i| * scale, plus that rounding again: joining the two halves of a group's sum is one rounding of
2^-24, scale * 2^-e exact, the row's sum one f32 step a group and at most 10 more between CTAs and for the bias.  A
group whose offset part (8 times the sum of x) cancels costs nothing: it is exact."""
import ctypes as C

import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu


def quantize4_numpy(w, group):
    """Codes and scales from the definition, each f32 operation as numpy's f32 (IEEE) and the rounding in 64 bits."""
    w = np.asarray(w, dtype=np.float32)
    n, k = w.shape
    groups = -(-k // group)
    codes, scales = np.zeros((n, k), np.int8), np.ones((n, groups), np.float32)
    with np.errstate(all="ignore"):
        for g in range(groups):
            part = w[:, g * group:(g + 1) * group]
            top = np.nanmax(np.where(np.isnan(part), np.float32(0), np.abs(part)), axis=1)
            scales[:, g] = np.where(top > 0, top / np.float32(7), np.float32(1))
            inv = np.float32(1) / scales[:, g]
            t = (part * inv[:, None]).astype(np.float32).astype(np.float64)
            r = np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -8, 7)
            codes[:, g * group:(g + 1) * group] = np.where(np.isnan(t), 0, r).astype(np.int8)
    return codes, scales


def pack4(codes):
    n, k = codes.shape
    c = np.zeros((n, k + k % 2), np.uint8)
    c[:, :k] = codes.astype(np.int16) & 15
    return c[:, 0::2] | (c[:, 1::2] << 4)


def exact(codes, scales, group, x, bias):
    """(y, bound) in 64 bits."""
    w = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), group, axis=1)[:, :codes.shape[1]]
    xd = x.astype(np.float64)
    y = xd @ w.T
    s = np.abs(xd) @ np.abs(w).T
    groups = scales.shape[1]
    floor = np.zeros_like(s)
    for g in range(groups):
        part = slice(g * group, (g + 1) * group)
        floor += np.abs(xd[:, part]).max(axis=1)[:, None] * np.abs(w[:, part]).sum(axis=1)[None, :]
    if bias is not None:
        y = y + bias
        s = s + np.abs(bias)
    bound = s * (groups + 12) * 2.0 ** -24 + floor * 2.0 ** -23 * 1.001
    return y, bound + 1e-37


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 31, 32), (5, 33, 64), (16, 64, 64), (17, 130, 128), (64, 4096, 128),
                                       (33, 1003, 32), (40, 264, 64), (7, 1000, 128), (300, 96, 32)])
def test_codes_and_scales_bit_for_bit(nne, ctx, n, k, group):
    w = oracle.normal(700, n * k + group, (n, k), 0.0, 0.02)
    w[0, 0] = 0.0
    if k > 8:
        w[-1, 3], w[-1, 5] = np.nan, -0.0
    if n > 2:
        w[1] = 0.0                                                     # an empty row: scale 1, codes 0
        w[2] = np.float32(3.5) * np.sign(oracle.normal(701, k, (k,)))  # halves: 3.5 / (3.5/7) = 7
    if n > 4:
        w[3, ::2] = np.float32(0.25)
        w[3, 0] = np.float32(3.5)                                      # 0.25 * 2 = 0.5 exactly: away from zero
        w[4] = np.float32(1e-44)                                       # the scale underflows
    codes, scales = quantize4_numpy(w, group)
    ql = nne.QLinear4.from_linear(nne.Linear(w), group, ctx)
    assert np.array_equal(ql.scales.view(np.uint32), scales.view(np.uint32))
    assert np.array_equal(ql.qweight, pack4(codes))
    want = codes.astype(np.float32) * np.repeat(scales, group, axis=1)[:, :k]
    assert np.array_equal(ql.to_linear().weight, want.astype(np.float32))


@pytest.mark.parametrize("offset", [0, 1])
def test_quantize_device_entry(nne, ctx, offset):
    """The device entry at an aligned and an unaligned base gives what the layer holds, and writes nothing else."""
    import torch
    n, k, group = 37, 520, 64
    w = oracle.normal(702, 0, (n, k), 0.0, 0.05)
    buf = torch.zeros(n * k + 8, device="cuda")
    buf[offset:offset + n * k] = torch.from_numpy(w.reshape(-1))
    q = torch.full((n * k // 2 + 64,), 0x5A, device="cuda", dtype=torch.uint8)
    s = torch.full((n * 9 + 8,), -3.0, device="cuda")
    nne.quantize_rows4_device(ctx, buf.data_ptr() + 4 * offset, n, k, group, q.data_ptr() + 4 * offset, s.data_ptr(),
                              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = quantize4_numpy(w, group)
    at = 4 * offset
    assert np.array_equal(q[at:at + n * k // 2].cpu().numpy().reshape(n, -1), pack4(codes))
    assert (q[:at] == 0x5A).all() and (q[at + n * k // 2:] == 0x5A).all()
    assert np.array_equal(s[:n * 9].cpu().numpy().reshape(n, 9), scales) and (s[n * 9:] == -3.0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,m", [(1, 1, 1), (5, 31, 2), (16, 64, 1), (129, 128, 3), (100, 1003, 5), (250, 4096, 1),
                                   (384, 2050, 9), (130, 700, 17), (70, 1500, 33), (4096, 512, 70), (130, 11008, 4),
                                   (130, 28672, 1), (33, 20000, 18)])
def test_forward(nne, ctx, n, k, m, group):
    codes, scales = quantize4_numpy(oracle.normal(703, n + k + group, (n, k), 0.0, 0.02), group)
    bias = oracle.normal(704, n, (n,), 0.0, 0.1) if n % 2 else None
    x = oracle.normal(705, m + k, (m, k))
    ql = nne.QLinear4.from_fields(pack4(codes), scales, bias, k, n, group, ctx)
    y = ql.forward(x)
    ref, bound = exact(codes, scales, group, x, bias)
    assert np.all(np.abs(y - ref) <= bound), float((np.abs(y - ref) / bound).max())
    assert np.array_equal(y, ql.forward(x))  # the order of sums is fixed


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,m", [(4743, 4100, 3), (37901, 70, 1), (5000, 4096, 4), (701, 2050, 12), (130, 9000, 11)])
def test_forward_of_large_layers(nne, ctx, n, k, m, group):
    """Layers whose blocks of 256 rows are enough for every SM, the last one ragged; and twelve rows in one pass."""
    codes, scales = quantize4_numpy(oracle.normal(717, n + k + group, (n, k), 0.0, 0.02), group)
    bias = oracle.normal(718, n, (n,), 0.0, 0.1)
    x = oracle.normal(719, m + k, (m, k))
    ql = nne.QLinear4.from_fields(pack4(codes), scales, bias, k, n, group, ctx)
    y = ql.forward(x)
    ref, bound = exact(codes, scales, group, x, bias)
    assert np.all(np.abs(y - ref) <= bound), float((np.abs(y - ref) / bound).max())
    assert np.array_equal(y, ql.forward(x))
    if m <= 4:
        assert np.array_equal(y[:1], ql.forward(x[:1]))


def test_wide_ranges_inside_a_row(nne, ctx):
    """Groups of very unlike size side by side, denormals and numbers near the end of f32."""
    n, k, group = 40, 256, 32
    codes, scales = quantize4_numpy(oracle.normal(706, 0, (n, k), 0.0, 0.02), group)
    x = oracle.normal(707, 0, (4, k))
    x *= np.repeat(np.array([1e-30, 1e30, 1.0, 1e-10, 1e10, 0.0, 1e20, 1e-20], np.float32), group)[None, :]
    x[1] = 1e-40
    x[2] = oracle.normal(708, 0, (k,)) * np.float32(1e36)
    ql = nne.QLinear4.from_fields(pack4(codes), scales, None, k, n, group, ctx)
    y = ql.forward(x)
    ref, bound = exact(codes, scales, group, x, None)
    bound[1] += 2.0 ** -149 * 8 * k  # a denormal row: one denormal step an element at most
    assert np.all(np.abs(y - ref) <= bound)


def test_inf_and_nan_stay_in_their_row(nne, ctx):
    n, k, group = 130, 300, 64
    codes, scales = quantize4_numpy(oracle.normal(709, 0, (n, k), 0.0, 0.02), group)
    x = oracle.normal(710, 0, (6, k))
    clean = x.copy()
    x[1, 7], x[4, 299] = np.inf, np.nan
    ql = nne.QLinear4.from_fields(pack4(codes), scales, None, k, n, group, ctx)
    y, z = ql.forward(x), ql.forward(clean)
    for r in (0, 2, 3, 5):
        assert np.array_equal(y[r], z[r])
    assert not np.isfinite(y[1]).any() and not np.isfinite(y[4]).any()


def test_strides_streams_and_capture(nne, ctx):
    """x at an address that is only 4-byte aligned, y as a slice of wider rows (the rest untouched), another stream
    than the default one, right behind the kernel that makes x; then captured and replayed on new inputs."""
    import torch
    n, k, m, group, ldy = 200, 512, 6, 64, 260
    codes, scales = quantize4_numpy(oracle.normal(711, 0, (n, k), 0.0, 0.02), group)
    ql = nne.QLinear4.from_fields(pack4(codes), scales, None, k, n, group, ctx)
    buf = torch.zeros(m * k + 4, device="cuda")
    y = torch.full((m, ldy), 7.0, device="cuda")
    src = torch.from_numpy(oracle.normal(712, 0, (m * k,))).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        buf[1:1 + m * k] = src * 2.0
        ql.forward_device(buf.data_ptr() + 4, m, y.data_ptr(), s.cuda_stream, ldy)
    s.synchronize()
    ref, bound = exact(codes, scales, group, (src.cpu().numpy() * 2).reshape(m, k), None)
    assert np.all(np.abs(y[:, :n].cpu().numpy() - ref) <= bound) and (y[:, n:] == 7.0).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        buf[1:1 + m * k] = src * 3.0
        ql.forward_device(buf.data_ptr() + 4, m, y.data_ptr(), s.cuda_stream, ldy)
    src.copy_(torch.from_numpy(oracle.normal(713, 0, (m * k,))))
    g.replay()
    torch.cuda.synchronize()
    ref, bound = exact(codes, scales, group, (src.cpu().numpy() * np.float32(3)).reshape(m, k), None)
    assert np.all(np.abs(y[:, :n].cpu().numpy() - ref) <= bound)


def test_rows_do_not_depend_on_their_neighbours(nne, ctx):
    n, k, group = 300, 1024, 32
    codes, scales = quantize4_numpy(oracle.normal(714, 0, (n, k), 0.0, 0.02), group)
    x = oracle.normal(715, 0, (32, k))
    ql = nne.QLinear4.from_fields(pack4(codes), scales, None, k, n, group, ctx)
    for lo, hi in ((1, 4), (5, 8), (9, 16), (17, 32)):
        assert np.array_equal(ql.forward(x[:lo]), ql.forward(x[:hi])[:lo])


def test_device_layer_and_empty_cases(nne, ctx):
    ql = nne.QLinear4.from_linear(nne.Linear(np.ones((4, 64), np.float32), np.arange(4, dtype=np.float32)), 32, ctx)
    assert ql.forward(np.zeros((0, 64), np.float32)).shape == (0, 4)
    x = nne.CudaTensor.from_raw(np.ones((2, 3, 64), np.float32), ctx)
    out = ql.to_gpu().forward(x)
    assert out.shape == [2, 3, 4] and np.array_equal(out.to_cpu(), np.broadcast_to(64 + np.arange(4, dtype=np.float32), (2, 3, 4)))
    empty = nne.QLinear4.from_fields(np.zeros((3, 0), np.uint8), np.zeros((3, 0), np.float32), np.array([1, 2, 3], np.float32), 0, 3, 64, ctx)
    assert np.array_equal(empty.forward(np.zeros((2, 0), np.float32)), np.array([[1, 2, 3]] * 2, np.float32))
    none = nne.QLinear4.from_fields(np.zeros((0, 4), np.uint8), np.zeros((0, 1), np.float32), None, 8, 0, 32, ctx)
    assert none.forward(np.zeros((2, 8), np.float32)).shape == (2, 0)
    assert ql.memory_bytes() == 16 * 64 // 2 + 16 * 2 * 4 + 4 * 4 and ql.parameters() == []


def test_layers_made_on_the_device_give_their_fields_back(nne, ctx):
    import torch
    n, k, group = 19, 77, 32
    w, bias = oracle.normal(716, 0, (n, k), 0.0, 0.02), oracle.normal(716, 1, (n,))
    wd, bd = torch.from_numpy(w).cuda(), torch.from_numpy(bias).cuda()
    s = torch.cuda.current_stream().cuda_stream
    codes, scales = quantize4_numpy(w, group)
    a = nne.QLinear4.from_linear_device(ctx, wd.data_ptr(), bd.data_ptr(), n, k, group, s)
    qd, sd = torch.from_numpy(pack4(codes)).cuda(), torch.from_numpy(scales).cuda()
    b = nne.QLinear4.from_packed_device(ctx, qd.data_ptr(), sd.data_ptr(), bd.data_ptr(), n, k, group, s)
    c = nne.QLinear4.from_packed_device(ctx, qd.data_ptr(), sd.data_ptr(), 0, n, k, group, s)
    for x in (a, b, c):
        assert np.array_equal(x.qweight, pack4(codes)) and np.array_equal(x.scales, scales)
    assert np.array_equal(a.bias, bias) and np.array_equal(b.to_linear().bias, bias) and c.bias is None
    with pytest.raises(nne.InvalidArgument):
        nne.QLinear4.from_packed_device(ctx, qd.data_ptr(), sd.data_ptr() + 2, 0, n, k, group, s)
    with pytest.raises(nne.InvalidArgument):
        nne.quantize_rows4_device(ctx, wd.data_ptr() + 1, 1, 4, group, qd.data_ptr(), sd.data_ptr(), s)


def test_refusals(nne, ctx):
    w = nne.Linear(np.ones((4, 64), np.float32))
    for group in (0, 16, 48, 256):
        with pytest.raises(nne.InvalidArgument):
            nne.QLinear4.from_linear(w, group, ctx)
    ql = nne.QLinear4.from_linear(w, 64, ctx)
    with pytest.raises(nne.InvalidArgument):
        ql.forward(np.zeros(64, np.float32))
    with pytest.raises(nne.ShapeMismatch):
        ql.forward(np.zeros((1, 65), np.float32))
    lib, one = nne.load(), C.c_void_p(16)
    assert lib.nne_qlinear4_forward_dev(ql._handle, one, 1, 63, one, None) == 2
    assert lib.nne_qlinear4_forward_dev_strided(ql._handle, one, 1, 64, one, 3, None) == 1
    assert lib.nne_qlinear4_forward_dev(ql._handle, None, 1, 64, one, None) == 1
    assert lib.nne_qlinear4_forward_dev(ql._handle, C.c_void_p(18), 1, 64, one, None) == 1
    assert lib.nne_qlinear4_forward_dev(ql._handle, one, 2 ** 60, 64, one, None) == 1
    ql.close()
    with pytest.raises(nne.GpuError):
        ql.forward_device(16, 1, 16)
