"""MATMUL_I4 on the GPU against products in 64 bits (serving_ops.py)."""
import ctypes as C

import numpy as np
import pytest

import serving_ops as ops
from vnpu_mi355x import Session, abi

pytestmark = pytest.mark.gpu


@pytest.fixture()
def own():
    """A session of its own: an error on a stream stays."""
    s = Session()
    yield s
    s.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def case(s, M, K, N, group, zeros=True, trans=False, bias=False, epilogue=0, a_gap=0, c_gap=0, shift=0, pad=0, seed=3, change=None,
         check=True):
    rng = np.random.default_rng(seed)
    w = ops.Weights(rng, K, N, group, zeros, trans, pad)
    a = normal(rng, M, K)
    a[:, rng.random(K) < 0.01] *= 30
    if change:
        change(a, w)
    b = normal(rng, N) if bias else None
    packed = w.pack(s)
    lda, ldc = K + a_gap, N + c_gap
    memory = np.full(shift + M * lda, np.nan, np.float32)   # what lies between the rows is not read
    memory[shift:].reshape(M, lda)[:, :K] = a
    ba, bc = s.upload(memory), s.upload(np.full((M, ldc), 7.0, np.float32))
    bb = s.upload(b) if bias else None
    s.run(abi.OP_MATMUL_I4, A=ba.ptr + 4 * shift, B=packed, C=bc, bias=bb, M=M, K=K, N=N, lda=lda if a_gap else 0,
          ldc=ldc if c_gap else 0, epilogue=epilogue)
    got = s.download(bc, np.float32, (M, ldc))
    for x in (ba, bc, bb):
        if x is not None:
            s.free(x)
    s.release_packed_i4(packed)
    assert np.all(got[:, N:] == 7.0)
    got = got[:, :N]
    if check:
        want, bound = ops.matmul(a, w, b, epilogue)
        off = np.abs(got - want)
        assert np.all(off <= bound), (float((off - bound).max()), np.argwhere(~(off <= bound))[:3].tolist())
        if K >= 64 and M * N >= 64 and not change and not epilogue:
            # Roundings of random signs: as many as the bound counts, of the result's size.
            assert np.sqrt(np.mean(off**2) / np.mean(want**2)) <= (4 + np.sqrt(K / 16 + 100)) * ops.EPS
    return got, a, w


ROWS = [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 128, 129, 200, 257]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("group", [32, 64, 128, 0])
def test_row_counts_and_groups(gpu, M, group):
    case(gpu, M, 640, 208, group, zeros=group != 64)


@pytest.mark.parametrize("M", [1, 6, 40, 150])
@pytest.mark.parametrize("K", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 192, 255, 257, 500, 1000, 1153])
def test_lengths_of_rows(gpu, M, K):
    for i, group in enumerate((32, 64, 128, 256, 0)):
        case(gpu, M, K, 33, group, zeros=(K + i) % 2 == 0, trans=(K + i) % 3 == 0)


@pytest.mark.parametrize("M", [1, 7, 30, 140])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 129, 255, 257, 1001])
def test_columns(gpu, M, N):
    case(gpu, M, 300, N, 64, trans=N % 2 == 0)
    case(gpu, M, 300, N, 128, zeros=False, trans=N % 2 == 1)


@pytest.mark.parametrize("M,K,N,group", [(1, 4096, 4096, 128), (1, 11008, 512, 64), (3, 4096, 32000, 128), (8, 11008, 4096, 64),
                                         (12, 8192, 1024, 32), (16, 4096, 2048, 0), (24, 4096, 4096, 128), (64, 2048, 8200, 32),
                                         (130, 4096, 1000, 384), (300, 1000, 4100, 64), (1100, 512, 520, 128), (2048, 256, 640, 32)])
def test_sizes_of_models(gpu, M, K, N, group):
    case(gpu, M, K, N, group)


@pytest.mark.parametrize("M,K,N", [
    (1, 2048, 48), (1, 16384, 16), (1, 2048, 6000), (1, 16384, 1001), (3, 64, 16), (3, 8192, 16), (2, 64, 11008), (2, 11008, 6000),
    (1, 300, 16001), (4, 8192, 2048), (5, 2048, 16), (7, 16384, 16), (8, 2048, 6000), (6, 16384, 1001), (5, 64, 17), (8, 4096, 16),
    (5, 100, 11008), (5, 64, 16000), (6, 4096, 2048), (9, 64, 16), (13, 2048, 16), (9, 64, 6000), (17, 4096, 500), (9, 64, 11008),
    (48, 4096, 1001), (17, 64, 8192), (17, 4096, 1001), (17, 64, 11008), (33, 2000, 11008), (17, 64, 16000), (19, 8192, 2048),
    (600, 64, 16), (601, 1000, 16), (600, 64, 4096), (601, 100, 6000), (600, 64, 11008), (600, 700, 300)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_kernel(gpu, M, K, N, group):
    """Sizes that between them take every kernel and cut, as test_serving_host has them."""
    case(gpu, M, K, N, group, zeros=group != 128, bias=N % 2 == 1)


@pytest.mark.parametrize("M", [1, 5, 20, 70, 130])
@pytest.mark.parametrize("epilogue", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("bias", [False, True])
def test_bias_and_epilogues(gpu, M, epilogue, bias):
    case(gpu, M, 200, 70, 32, bias=bias, epilogue=epilogue)


@pytest.mark.parametrize("M,K", [(1, 40), (3, 8192), (12, 40), (20, 8192), (600, 40)])
@pytest.mark.parametrize("epilogue", [abi.EPI_SILU, abi.EPI_GELU_TANH, abi.EPI_GELU_ERF])
def test_epilogues_to_a_part_of_the_result(gpu, M, K, epilogue):
    """Of the bias alone, A being zero.  To a part of the result, down its left tail too: an exponential is off by 2^-23 at most (1
    ulp), and there are four roundings of 2^-24 beside it, one more for GELU_TANH: together below 2^-21.  erfc may be off by
    2^-19 (16 ulp, what OpenCL allows a device library).  An exponential or erfc in steps of 2^-149, times x up to 104, is
    2^-142."""
    x = np.concatenate([-np.geomspace(104, 1e-30, 3000), np.linspace(-16, 16, 3001), np.geomspace(1e-30, 1e30, 1000), [0.0, -1e4, -1e30]])
    x = x.astype(np.float32)
    N = x.size
    w = ops.Weights(np.random.default_rng(2), K, N, 0)
    packed = w.pack(gpu)
    ba, bb, bc = gpu.upload(np.zeros((M, K), np.float32)), gpu.upload(x), gpu.alloc(4 * M * N)
    gpu.run(abi.OP_MATMUL_I4, A=ba, B=packed, C=bc, bias=bb, M=M, K=K, N=N, epilogue=epilogue)
    got = gpu.download(bc, np.float32, (M, N))
    for b in (ba, bb, bc):
        gpu.free(b)
    gpu.release_packed_i4(packed)
    with np.errstate(over="ignore"):
        want = ops.finished(x.astype(np.float64), epilogue)
    part = 2.0**-21 + (2.0**-19 if epilogue == abi.EPI_GELU_ERF else 0)
    off = np.abs(got - want) / (part * np.abs(want) + 2.0**-142)
    assert np.all(off <= 1), [(float(x[i]), float(got[r, i]), float(want[i])) for r, i in np.argwhere(~(off <= 1))[:5]]


@pytest.mark.parametrize("M", [1, 4, 19, 66, 131])
@pytest.mark.parametrize("a_gap,c_gap,shift,pad", [(4, 0, 0, 0), (1, 3, 0, 0), (0, 5, 1, 3), (3, 1, 2, 0), (8, 4, 4, 1), (0, 0, 3, 16)])
def test_strides_and_alignment(gpu, M, a_gap, c_gap, shift, pad):
    case(gpu, M, 260, 50, 64, a_gap=a_gap, c_gap=c_gap, shift=shift, pad=pad)
    case(gpu, M, 257, 51, 32, a_gap=a_gap, c_gap=c_gap, shift=shift, pad=pad, trans=True)


@pytest.mark.parametrize("M", [2, 12, 40, 140])
@pytest.mark.parametrize("factor", [1e-44, 1e-38, 1e-30, 1e-20, 1e20, 1e34])
def test_sizes_of_values(gpu, M, factor):
    """Rows at the ends of f32, one of them zero."""
    def change(a, w):
        a *= np.float32(factor)
        a[1] = 0
    with np.errstate(under="ignore", over="ignore"):
        case(gpu, M, 200, 40, 64, change=change)


@pytest.mark.parametrize("M", [1, 4, 8, 12, 40, 140])
@pytest.mark.parametrize("power", [-97, -96, -95, -88, -80, -64])
@pytest.mark.parametrize("scale", [1e-3, 1e-5, 1e-7])
def test_small_values_with_small_scales(gpu, M, power, scale):
    """A row's power of two and a scale whose product is no normal number; the results are."""
    def change(a, w):
        a *= np.float32(2.0**power / 8)
        w.scales *= np.float32(scale / 0.02)
    for group in (32, 64, 128):
        case(gpu, M, 260, 40, group, zeros=group != 128, change=change)


@pytest.mark.parametrize("M", [1, 4, 8, 12, 40, 140])
@pytest.mark.parametrize("power,scale", [(-96, 1e17), (-70, 1e17), (-96, 1e25), (-20, 1e-25), (0, 1e-30), (60, 1e-34), (100, 1e-30)])
def test_values_and_scales_at_opposite_ends(gpu, M, power, scale):
    """A sum in a row's own unit, or that unit, times a scale is beyond the normal numbers; the results are not."""
    def change(a, w):
        a *= np.float32(2.0**power / 8)
        w.scales *= np.float32(scale / 0.02)
    for group in (32, 64, 128):
        case(gpu, M, 260, 40, group, zeros=group != 128, change=change)


@pytest.mark.parametrize("M", [3, 14, 40, 140])
def test_values_far_apart(gpu, M):
    """A row whose largest element is 2^60 times the others, in a block of its own and among them."""
    def change(a, w):
        a[0, 5] = 2.0**60
        a[1, 200:] *= np.float32(2.0**-60)
        a[2, 130] = -(2.0**30)
    case(gpu, M, 384, 40, 128, change=change)


@pytest.mark.parametrize("M", [4, 15, 40, 140])
def test_not_finite(gpu, M):
    """A row with an infinity or NaN gives NaN, others do not see it; a scale that is none gives NaN in its column."""
    def change(a, w):
        a[1, 3], a[2, 199] = np.nan, -np.inf
        w.scales[1, 7] = np.nan
    got, a, w = case(gpu, M, 200, 40, 64, change=change, check=False)
    want = np.zeros(got.shape, bool)
    want[1:3] = True
    want[:, 7] = True
    assert np.array_equal(np.isnan(got), want)


@pytest.mark.parametrize("M", [1, 3, 8, 9, 20, 40])
@pytest.mark.parametrize("K", [1, 100, 129, 700, 1100, 2100])
@pytest.mark.parametrize("N", [16, 33, 49, 80, 1000])
def test_waves_without_blocks_and_strips_behind_the_last(gpu, M, K, N):
    """What lies behind a range of blocks or the last strip, and a last scale that is none, changes nothing else."""
    for group in (32, 64, 256):
        def change(a, w):
            w.scales[-1, N - 1] = np.nan
        got, a, w = case(gpu, M, K, N, group, zeros=group != 64, change=change, check=False)
        assert np.all(np.isnan(got[:, N - 1]))
        w.scales[-1, N - 1] = 0
        want, bound = ops.matmul(a, w)
        assert np.all(np.abs(got - want)[:, :N - 1] <= bound[:, :N - 1])


@pytest.mark.parametrize("M", [1, 3, 9, 40, 140])
def test_extreme_codes_and_signs(gpu, M):
    """Every product at its largest: 15 less zero of either sign, rows of one value."""
    for zero, code in ((0, 15), (15, 0), (15, 15), (0, 0), (8, 15)):
        def change(a, w):
            a[:] = np.where(np.arange(M)[:, None] % 2, -1.5, 1.999)
            w.codes[:] = code
            w.bytes[:] = code * 17
            w.zeros[:] = zero
        case(gpu, M, 1024, 20, 128, change=change)


@pytest.mark.parametrize("M", [1, 37])
def test_host_memory(own, M):
    rng = np.random.default_rng(1)
    w = ops.Weights(rng, 150, 45, 32)
    a, bias, out = normal(rng, M, 150), normal(rng, 45), np.full((M, 50), 7, np.float32)
    packed = w.pack(own)
    own.run(abi.OP_MATMUL_I4, A=a.ctypes.data, B=packed, bias=bias.ctypes.data, C=out.ctypes.data, M=M, K=150, N=45, ldc=50)
    want, bound = ops.matmul(a, w, bias)
    assert np.all(np.abs(out[:, :45] - want) <= bound) and np.all(out[:, 45:] == 7)


def test_packing_from_the_device_and_info(gpu):
    rng = np.random.default_rng(2)
    for trans in (False, True):
        w = ops.Weights(rng, 130, 37, 64, trans=trans, pad=2)
        bufs = [gpu.upload(x) for x in (w.bytes, w.scales, w.zeros)]
        p = gpu.pack_i4(bufs[0], bufs[1], w.K, w.N, 64, zeros=bufs[2], ldb=w.ldb, trans_b=int(trans))
        K, N, group, nbytes = C.c_uint32(), C.c_uint32(), C.c_uint32(), C.c_uint64()
        assert gpu.lib.vnpu_packed_weights_i4_info(p, C.byref(K), C.byref(N), C.byref(group), C.byref(nbytes)) == abi.OK
        assert (K.value, N.value, group.value) == (130, 37, 64) and nbytes.value >= 65 * 37
        a = normal(rng, 3, 130)
        ba, bc = gpu.upload(a), gpu.alloc(3 * 37 * 4)
        gpu.run(abi.OP_MATMUL_I4, A=ba, B=p, C=bc, M=3, K=130, N=37)
        want, bound = ops.matmul(a, w)
        assert np.all(np.abs(gpu.download(bc, np.float32, (3, 37)) - want) <= bound)
        gpu.release_packed_i4(p)
        for x in (*bufs, ba, bc):
            gpu.free(x)


@pytest.mark.parametrize("group", [384, 4096, 1 << 31, 0xffffff80])
def test_groups_of_more_than_a_column(gpu, group):
    """They are one group, however large."""
    for M in (1, 10, 40):
        got, a, w = case(gpu, M, 300, 40, 0)
        w.group = group
        packed, size = w.pack(gpu), C.c_uint32()
        assert gpu.lib.vnpu_packed_weights_i4_info(packed, None, None, C.byref(size), None) == abi.OK and size.value == group
        ba, bc = gpu.upload(a), gpu.alloc(4 * M * 40)
        gpu.run(abi.OP_MATMUL_I4, A=ba, B=packed, C=bc, M=M, K=300, N=40)
        assert np.array_equal(gpu.download(bc, np.float32, (M, 40)), got)
        gpu.release_packed_i4(packed)
        gpu.free(ba)
        gpu.free(bc)


def test_bad_weights_are_refused(gpu):
    codes, scales, out = np.zeros((64, 8), np.uint8), np.ones((2, 16), np.float32), C.c_void_p()
    zeros = np.full((2, 16), 15, np.uint8)

    def pack(K=64, N=16, group=32, ldb=0, trans=0, z=zeros, codes=codes.ctypes.data, scales=scales.ctypes.data):
        return gpu.lib.vnpu_pack_weights_i4(gpu.dev, codes, scales, z.ctypes.data, K, N, group, ldb, trans, C.byref(out))

    assert pack() == abi.OK
    gpu.lib.vnpu_packed_weights_i4_destroy(out)
    bad = zeros.copy()
    bad[1, 3] = 16
    for rc in (pack(z=bad), pack(K=0), pack(N=0), pack(group=16), pack(group=96), pack(group=192), pack(ldb=7), pack(trans=2),
               pack(codes=None), pack(scales=None), pack(K=(1 << 30) + 1), pack(K=1 << 30, N=1 << 20)):
        assert rc == abi.ERR_INVALID_ARGUMENT and not out.value


def test_refused_products_fail_the_stream(own):
    rng = np.random.default_rng(1)
    packed = ops.Weights(rng, 64, 32, 32).pack(own)
    a, c = own.alloc(64 * 4), own.upload(np.full(32, 7, np.float32))
    f = dict(A=a, B=packed, C=c, M=1, K=64, N=32)
    own.run(abi.OP_MATMUL_I4, **f)
    own.write(c, np.full(32, 7, np.float32))
    for bad in (dict(K=63), dict(N=31), dict(lda=60), dict(epilogue=9)):
        s = Session()
        try:
            p = ops.Weights(rng, 64, 32, 32).pack(s)
            assert s.submit([s.command(abi.OP_MATMUL_I4, **{**f, "B": p, **bad})]) == abi.OK
            assert s.sync() == abi.ERR_DEVICE_ERROR
        finally:
            s.close()
    assert np.all(own.download(c, np.float32, (32,)) == 7)


def test_the_same_call_gives_the_same_bits(gpu):
    for M, K, N in ((1, 4096, 1000), (8, 3000, 500), (40, 4096, 300), (200, 1000, 700)):
        first, *_ = case(gpu, M, K, N, 128)
        for _ in range(3):
            again, *_ = case(gpu, M, K, N, 128, check=False)
            assert np.array_equal(first, again)


def test_codes_beyond_32_bits_of_elements(gpu):
    """4 GiB elements of K x N: 2 GiB of codes; columns at either end against the definition."""
    K, N = 1 << 15, (1 << 17) + 16
    codes = gpu.alloc(N * K // 2)
    rng = np.random.default_rng(5)
    edge = rng.integers(0, 256, (16, K // 2)).astype(np.uint8)
    for n in (0, 1 << 16, N - 16):
        gpu.write(codes, edge, offset=n * (K // 2))
    scales = gpu.upload(np.ones((1, N), np.float32))
    p = gpu.pack_i4(codes, scales, K, N, 0, trans_b=1)
    gpu.free(codes)
    value = np.empty((16, K))
    value[:, 0::2], value[:, 1::2] = edge & 15, edge >> 4
    for M in (2, 70):
        a = normal(rng, M, K)
        ba, bc = gpu.upload(a), gpu.alloc(M * N * 4)
        gpu.run(abi.OP_MATMUL_I4, A=ba, B=p, C=bc, M=M, K=K, N=N)
        got = gpu.download(bc, np.float32, (M, N))
        want = a.astype(np.float64) @ (value.T - 8)
        bound = (2.0**-23 + (K / 16 + 100) * ops.EPS) * (np.abs(a).astype(np.float64) @ np.abs(value.T - 8))
        for n in (0, 1 << 16, N - 16):
            assert np.all(np.abs(got[:, n:n + 16] - want) <= bound)
        gpu.free(ba)
        gpu.free(bc)
    gpu.release_packed_i4(p)
    gpu.free(scales)
