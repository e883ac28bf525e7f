"""The projection's tiles of 128 and 256 results a side, in the forward and both gradients: whole and cut along the contraction, of one
stage (128 bytes of contraction), two, three and many, no dimension a multiple of anything. Every case names the product that it is
there for and how the library has to cut it, asked through gs_linear_plan, so that a rule that chooses other tiles shows. Values
are held to the bounds of test_gpu_linear.py, against float64."""
import ctypes as C
import math

import pytest
import torch

import test_gpu_linear as L
from amdsplat import _lib

BF16, F32 = torch.bfloat16, torch.float32
FORWARD, D_X, D_WEIGHT = range(3)

# type, product, side of the tiles, whole ones?, others in parts?, stages, (rows, outputs, inputs), activation
CASES = [
    (BF16, FORWARD, 256, True, False, 1, (1605, 8777, 51), "none"),
    (BF16, FORWARD, 256, True, False, 2, (1235, 9911, 81), "none"),
    (BF16, FORWARD, 256, True, False, 3, (3399, 3603, 165), "none"),
    (BF16, FORWARD, 256, True, False, 5, (10009, 1167, 307), "none"),
    (BF16, FORWARD, 256, False, True, 108, (3511, 2999, 6901), "gelu"),
    (BF16, FORWARD, 256, True, True, 57, (3223, 6441, 3629), "silu"),
    (BF16, D_X, 256, True, False, 1, (5889, 43, 2433), "gelu"),
    (BF16, D_X, 256, True, False, 2, (1557, 81, 7823), "none"),
    (BF16, D_X, 256, True, False, 3, (1219, 147, 9819), "relu"),
    (BF16, D_X, 256, True, False, 6, (9099, 361, 1285), "gelu_tanh"),
    (BF16, D_X, 256, False, True, 111, (3375, 7061, 3043), "none"),
    (BF16, D_X, 256, True, True, 59, (4771, 3771, 3499), "gelu"),
    (BF16, D_WEIGHT, 256, True, False, 1, (23, 9609, 1493), "none"),
    (BF16, D_WEIGHT, 256, True, False, 2, (71, 1241, 9815), "silu"),
    (BF16, D_WEIGHT, 256, True, False, 5, (269, 1165, 9841), "gelu"),
    (BF16, D_WEIGHT, 256, False, True, 102, (6499, 4131, 2525), "none"),
    (BF16, D_WEIGHT, 256, True, True, 58, (3675, 3985, 4777), "none"),
    (BF16, FORWARD, 128, True, False, 1, (8431, 323, 21), "gelu"),
    (BF16, FORWARD, 128, True, False, 2, (10053, 265, 75), "silu"),
    (BF16, FORWARD, 128, False, True, 57, (841, 1153, 3643), "gelu"),
    (BF16, FORWARD, 128, True, True, 20, (1233, 3305, 1231), "relu"),
    (BF16, D_X, 128, True, False, 4, (263, 197, 9895), "none"),
    (BF16, D_X, 128, False, True, 62, (991, 3919, 1025), "gelu"),
    (BF16, D_X, 128, True, True, 25, (2305, 1565, 1801), "none"),
    (BF16, D_WEIGHT, 128, True, False, 4, (195, 9913, 269), "none"),
    (BF16, D_WEIGHT, 128, False, True, 70, (4417, 1047, 971), "gelu"),
    (BF16, D_WEIGHT, 128, True, True, 20, (1233, 3305, 1231), "none"),
    (F32, FORWARD, 128, True, False, 1, (8941, 781, 23), "gelu"),
    (F32, FORWARD, 128, True, False, 2, (8251, 835, 59), "silu"),
    (F32, FORWARD, 128, False, True, 102, (1201, 939, 3241), "gelu"),
    (F32, FORWARD, 128, True, True, 33, (1299, 3493, 1027), "none"),
    (F32, D_X, 128, True, False, 2, (919, 63, 7619), "gelu"),
    (F32, D_X, 128, False, True, 84, (1519, 2673, 745), "none"),
    (F32, D_X, 128, True, True, 30, (3691, 943, 1217), "gelu_tanh"),
    (F32, D_WEIGHT, 128, True, False, 8, (237, 769, 8853), "none"),
    (F32, D_WEIGHT, 128, False, True, 102, (3247, 1347, 831), "gelu"),
    (F32, D_WEIGHT, 128, True, True, 31, (969, 1347, 3373), "none"),
]
KIND = {BF16: _lib.GS_BFLOAT16, F32: _lib.GS_FLOAT32}


def plan(dtype, product, shape, act, residual=None):
    """Side, whole tiles and parts of the others in a trained call with a bias."""
    m, n, k = shape
    ld = -(-k // 8) * 8
    a = _lib.GsLinear(x=256, weight=256, bias=256, out=256, z=256 if act != "none" else None, rows=m, x_stride=ld, weight_stride=ld,
                      residual=residual and 256, residual_stride=n, inputs=k, outputs=n, dtype=KIND[dtype],
                      out_dtype=KIND[residual or dtype], activation=L.ACTS.index(act))
    got = [C.c_int32(-1) for _ in range(3)]
    assert _lib.lib().gs_linear_plan(C.byref(a), product, *map(C.byref, got)) == 0
    return [v.value for v in got]


def names(c):
    return f"{'bf16' if c[0] == BF16 else 'f32'}-{('forward', 'd_x', 'd_weight')[c[1]]}-{c[2]}-{c[3]:d}{c[4]:d}-{c[5]}"


@pytest.mark.parametrize("case", CASES, ids=names)
def test_plans(case):
    dtype, product, side, whole, cut, stages, shape, act = case
    tile, alone, parts = plan(dtype, product, shape, act)
    assert (tile, alone > 0, parts > 0) == (side, whole, cut)
    along = (shape[2], shape[1], shape[0])[product]
    assert -(-along // (128 // dtype.itemsize)) == stages
    assert all(v % 2 for v in shape)


def test_plan_calls():
    lib = _lib.lib()
    a = _lib.GsLinear(x=256, weight=256, out=256, rows=16, x_stride=64, weight_stride=64, inputs=64, outputs=40)
    v = [C.c_int32(-1) for _ in range(3)]
    call = lambda a=a, product=0, v=v: lib.gs_linear_plan(a and C.byref(a), product, *[x and C.byref(x) for x in v])  # noqa: E731
    assert call() == 0 and [x.value for x in v] == [0, 0, 0]  # few rows
    for kw, text in ((dict(a=None), "NULL"), (dict(product=3), "product"), (dict(product=-1), "product"), (dict(v=[v[0], None, v[2]]), "null")):
        assert call(**kw) == 1 and text in lib.gs_last_error().decode()
    a.rows = 0
    assert call(product=D_X) == 0 and v[0].value == 0
    assert call(product=D_WEIGHT) == 0 and [x.value for x in v] == [64, 1, 0]


def tensors(seed, dtype, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return rand(m, k).to(dtype), (rand(n, k) / math.sqrt(k)).to(dtype), rand(n)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=names)
def test_tiles(case):
    dtype, product, side, whole, cut, _, shape, act = case
    tile, alone, parts = plan(dtype, product, shape, act)
    assert (tile, alone > 0, parts > 0) == (side, whole, cut)
    L.check(*tensors(5, dtype, *shape), act)


VIEWS = [  # type, the residual's, side of the tiles, whole ones?, others in parts?
    (BF16, BF16, 256, True, False, (10051, 1155, 1000)),
    (BF16, F32, 256, True, False, (3377, 3585, 1424)),
    (BF16, F32, 256, True, True, (5085, 3279, 3344)),
    (BF16, F32, 128, True, False, (265, 9853, 56)),
    (F32, F32, 128, False, True, (1263, 785, 1552)),
    (F32, F32, 128, True, True, (1347, 3381, 928)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,residual,side,whole,cut,shape", VIEWS)
def test_views_with_a_residual(dtype, residual, side, whole, cut, shape):
    """Views of wider tensors that hold NaN everywhere else: nothing of it is read into results."""
    m, n, k = shape
    tile, alone, parts = plan(dtype, FORWARD, shape, "none", residual)
    assert (tile, alone > 0, parts > 0) == (side, whole, cut)
    x, w, b = tensors(6, dtype, *shape)
    wide = lambda t: torch.full((t.shape[0] + 70, k + 24), math.nan, dtype=dtype, device="cuda")  # noqa: E731
    big, weights = wide(x), wide(w)
    big[:m, 8:k + 8], weights[:n, 16:k + 16] = x, w
    r = torch.full((m + 1, n + 5), math.nan, dtype=residual, device="cuda")
    r[:m, 3:n + 3] = tensors(7, residual, m, 1, n)[0]
    L.check(big[:m, 8:k + 8], weights[:n, 16:k + 16], b, "none", r[:m, 3:n + 3])
