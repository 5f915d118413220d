"""Sizes that reach each kernel of ops.linear and ops.window_attention, with the
form that the library's own host queries give for them."""
import ctypes

from dfsattn_amd import _lib, ops

# dfs_linear_form and dfs_window_attention_form
FEW, ANY, T64, T64X128, T128_DEEP, T128, T256 = range(7)
BLOCKS = 1
PARTS, STREAM, LAID_OUT, WIDE, SHORT_LAST = 16, 32, 64, 128, 256

# rows, outputs, channels, form: rows and outputs off every tile, the last
# channels no whole step, rows on 16-byte boundaries where channels are a
# multiple of 8
LINEAR = [
    (1, 77, 8, FEW | WIDE),
    (7, 1003, 520, FEW | WIDE),
    (5, 4105, 264, FEW),
    (8, 5003, 136, FEW),
    (3, 16411, 8264, FEW | STREAM),
    (2, 333, 1501, FEW | WIDE | LAID_OUT),
    (7, 4203, 1101, FEW | LAID_OUT),
    (1, 16411, 8251, FEW | STREAM | LAID_OUT),
    (131, 259, 709, ANY),
    (9, 65, 1, ANY),
    (77, 331, 328, T64),
    (33, 523, 2104, T64 | PARTS),
    (77, 331, 1101, T64 | LAID_OUT),
    (33, 523, 2101, T64 | PARTS | LAID_OUT),
    (131, 5627, 264, T64X128),
    (2049, 67, 2472, T64X128 | PARTS),
    (5685, 129, 1037, T64X128 | LAID_OUT),
    (2049, 67, 2477, T64X128 | PARTS | LAID_OUT),
    (1025, 2051, 328, T128_DEEP),
    (131, 5459, 7776, T128_DEEP | PARTS),
    (1975, 1147, 474, T128_DEEP | LAID_OUT),
    (5593, 137, 6892, T128_DEEP | PARTS | LAID_OUT),
    (1999, 2051, 1336, T128),
    (129, 5696, 7968, T128 | PARTS),
    (2989, 1400, 258, T128 | LAID_OUT),
    (4121, 204, 6799, T128 | PARTS | LAID_OUT),
    (4185, 1953, 264, T256),
    (4099, 5003, 200, T256),
    (2953, 5544, 1176, T256 | PARTS),
    (5385, 1426, 262, T256 | LAID_OUT),
    (3201, 4995, 1199, T256 | PARTS | LAID_OUT),
]


def linear_form(m, n, k, aligned=None):
    return _lib.lib().dfs_linear_form(m, n, k, int(k % 8 == 0 if aligned is None else aligned))


# batch, heads, key heads, queries, slots, head dim, left, right, sinks, rolling, form
WINDOW = [
    (2, 4, 2, 1, 90, 64, None, 0, 0, False, FEW),
    (1, 4, 2, 9, 1300, 128, None, None, 0, False, FEW | PARTS),
    (64, 20, 20, 1, 4200, 64, None, 0, 0, False, FEW | STREAM),
    (16, 16, 8, 1, 4200, 128, 4150, 0, 9, False, FEW | PARTS | STREAM),
    (16, 8, 8, 2, 4200, 128, 4101, None, 64, True, FEW | PARTS | STREAM),
    (32, 8, 8, 3, 4200, 64, 4190, 0, 4, True, FEW | PARTS | STREAM),
    (1, 3, 3, 150, 160, 64, 40, 3, 2, False, BLOCKS),
    (1, 2, 1, 130, 2600, 128, None, 0, 0, False, BLOCKS | PARTS),
    (1, 8, 8, 150, 300, 128, 50, 0, 4, False, BLOCKS | SHORT_LAST),
    (1, 8, 8, 150, 2000, 64, 1700, None, 64, True, BLOCKS | PARTS | SHORT_LAST),
]


def window_form(B, H, G, L, S, D, left, right, sinks, rolling, dtype):
    def strides(*shape):
        return ops._contiguous_stride(shape)

    q, k = (B, H, L, D), (B, G, S, D)
    head = ops._window_plan(q, strides(*q), k, strides(*k), k, strides(*k), (dtype,) * 3, None, left, right, sinks,
                            rolling, rolling, None)[0]
    block = head + bytes(ctypes.sizeof(_lib.WindowArgs) - len(head))
    return _lib.lib().dfs_window_attention_form(block)
