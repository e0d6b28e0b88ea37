"""Products whose kernels the smaller tests do not reach, and what is planned for
each (not collected by pytest): type, out, inp, cols, the side that W lies along,
groups, elements between columns, activation; then for the product, dX and dW the
sums a workgroup makes (rows, columns), whether its operands are copied to LDS, the
pieces of k, and what is packed first (1 W, 2 X, 4 dY).  No extent is a whole number
of tiles."""
import ctypes

from jlust_amd import _lib, layers
from jlust_amd.elementwise import FN_GELU, FN_IDENTITY, FN_RELU, FN_SILU

ACTS = {None: FN_IDENTITY, "relu": FN_RELU, "gelu": FN_GELU, "silu": FN_SILU}
TYPES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3}

PLANNED = [
    ("bf16", 2053, 200, 14600, "out", 0, 0, "gelu", (256, 256, 1, 1, 1), (128, 128, 0, 1, 4), (256, 128, 1, 8, 4)),
    ("f16", 2104, 200, 14600, "inp", 0, 0, None, (256, 256, 1, 1, 0), (128, 128, 1, 1, 0), (256, 128, 1, 8, 0)),
    ("bf16", 2104, 200, 14600, "inp", 3, 0, "silu", (256, 256, 1, 1, 0), (128, 128, 1, 1, 4), (256, 128, 1, 4, 6)),
    ("f16", 2053, 201, 14600, "out", 3, 0, None, (256, 256, 1, 1, 3), (128, 128, 0, 1, 4), (256, 128, 1, 4, 6)),
    ("bf16", 200, 2053, 14600, "out", 0, 0, None, (128, 128, 0, 1, 0), (256, 256, 1, 1, 0), (64, 64, 0, 8, 0)),
    ("f16", 200, 2104, 14600, "inp", 3, 0, None, (128, 128, 1, 1, 0), (256, 256, 1, 1, 4), (256, 128, 1, 4, 6)),
    ("bf16", 201, 2053, 14600, "inp", 0, 0, "relu", (128, 128, 0, 1, 0), (256, 256, 1, 1, 5), (64, 64, 0, 8, 4)),
    ("f16", 264, 200, 14600, "inp", 0, 0, "gelu", (256, 128, 1, 1, 0), (128, 128, 1, 1, 4), (128, 128, 1, 32, 4)),
    ("bf16", 264, 200, 14600, "out", 3, 0, None, (256, 128, 1, 1, 0), (128, 128, 1, 1, 4), (64, 64, 0, 8, 6)),
    ("bf16", 200, 264, 14600, "out", 3, 0, None, (128, 128, 1, 1, 0), (256, 128, 1, 1, 4), (64, 64, 0, 8, 6)),
    ("bf16", 1000, 2104, 300, "out", 0, 0, None, (128, 128, 1, 8, 0), (64, 64, 0, 1, 0), (128, 128, 1, 1, 0)),
    ("f16", 200, 520, 2050, "out", 0, 0, None, (64, 64, 0, 1, 0), (64, 64, 0, 1, 0), (128, 128, 1, 16, 0)),
    ("bf16", 1544, 2053, 1200, "inp", 0, 0, None, (64, 64, 0, 1, 0), (64, 64, 0, 1, 0), (128, 128, 1, 1, 2)),
    ("f16", 1000, 4104, 300, "inp", 0, 0, "gelu", (128, 128, 1, 8, 0), (64, 64, 0, 1, 4), (256, 128, 1, 1, 4)),
    ("bf16", 4104, 1001, 600, "out", 0, 0, None, (64, 64, 0, 1, 0), (128, 128, 1, 4, 0), (256, 128, 1, 1, 2)),
    ("f16", 1531, 2053, 40, "inp", 0, 0, None, (128, 32, 0, 8, 0), (128, 32, 0, 8, 0), (128, 128, 0, 1, 0)),
    ("bf16", 201, 4001, 4100, "inp", 0, 0, None, (64, 64, 0, 4, 0), (128, 128, 1, 1, 5), (128, 128, 0, 4, 4)),
    ("f16", 1029, 200, 40, "out", 3, 0, "silu", (32, 16, 0, 1, 0), (16, 16, 0, 1, 4), (64, 64, 0, 1, 6)),
    ("bf16", 1029, 200, 40, "out", 3, 0, None, (32, 16, 0, 1, 0), (16, 16, 0, 1, 4), (64, 64, 0, 1, 6)),
    ("bf16", 520, 2104, 150, "inp", 3, 0, "gelu", (128, 128, 1, 16, 0), (64, 64, 0, 1, 4), (128, 128, 0, 1, 6)),
    ("f32", 1544, 264, 2050, "out", 0, 0, "gelu", (128, 128, 1, 1, 0), (96, 64, 0, 2, 4), (64, 64, 0, 4, 4)),
    ("f32", 1544, 264, 2050, "inp", 3, 0, None, (128, 128, 1, 1, 0), (96, 64, 0, 2, 4), (64, 64, 0, 1, 6)),
    ("f32", 264, 1531, 2050, "out", 3, 0, None, (96, 64, 0, 2, 0), (128, 128, 1, 1, 4), (64, 64, 0, 1, 6)),
    ("f32", 264, 1544, 8200, "inp", 3, 1, "silu", (96, 64, 0, 1, 0), (128, 128, 1, 1, 5), (64, 64, 0, 2, 6)),
    ("f32", 1531, 264, 4100, "out", 0, 0, None, (128, 128, 1, 1, 1), (96, 64, 0, 1, 0), (64, 64, 0, 4, 0)),
    ("f32", 4104, 333, 1200, "out", 0, 0, None, (128, 128, 1, 1, 2), (112, 64, 0, 4, 0), (64, 64, 0, 1, 2)),
    ("f32", 333, 4104, 1200, "inp", 0, 0, "relu", (112, 64, 0, 4, 0), (128, 128, 1, 1, 4), (64, 64, 0, 1, 4)),
    ("f32", 1544, 264, 14600, "inp", 0, 1, None, (128, 128, 1, 1, 3), (96, 64, 0, 1, 1), (64, 64, 0, 4, 2)),
    ("f32", 1000, 4104, 40, "out", 0, 1, None, (128, 32, 0, 16, 0), (128, 32, 0, 2, 0), (128, 128, 0, 1, 0)),
    ("f32", 1544, 4104, 100, "out", 0, 0, None, (128, 128, 1, 16, 0), (64, 64, 0, 4, 0), (128, 128, 1, 1, 0)),
    ("f32", 4104, 1544, 100, "out", 0, 0, "gelu", (64, 64, 0, 4, 0), (128, 128, 1, 16, 4), (128, 128, 1, 1, 4)),
    ("f32", 200, 520, 4100, "out", 3, 0, None, (112, 64, 0, 1, 0), (112, 64, 0, 1, 4), (128, 128, 1, 8, 6)),
    ("f32", 200, 200, 14600, "out", 0, 0, None, (112, 64, 0, 1, 0), (112, 64, 0, 1, 0), (128, 128, 1, 64, 0)),
]


def info(packed, grad=False):
    """jlust_hip_linear_info, or _grad_info's two, of packed arguments."""
    r = (ctypes.c_int64 * 12)()
    f = _lib.lib().jlust_hip_linear_grad_info if grad else _lib.lib().jlust_hip_linear_info
    _lib.check(f(packed, r), "linear_info")
    return (tuple(r[:6]), tuple(r[6:])) if grad else tuple(r[:6])


def arguments(T, out, inp, cols, layout, groups, pad, act):
    """The packed arguments of both calls: operands at aligned addresses, their columns
    `pad` elements apart but for those that a gradient call brings (dY, dX, dW)."""
    T, p = TYPES[T], 1 << 20
    a, b = (out, inp) if layout == "out" else (inp, out)
    head = (T, ACTS[act], int(layout == "inp"), 0, out, inp, cols, p, a + pad, p, inp + pad, p)
    tail = (groups, 1, p if groups else 0, (a + pad) * b)
    z = (p, out + pad) if act else (0, 0)
    return (layers._LINEAR(*head, out + pad, 0, 0, 0, 0, 0, *tail, 0),
            layers._LINEAR_GRAD(*head, out, *z, p, inp, p, a, 0, *tail, a * b, 0))
