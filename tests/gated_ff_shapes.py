"""Sizes that the gated feed-forward product takes through each of its tile paths: {(rows,
d, ff): [(which, tile, cuts of dx, cuts of dW, whether a CTA or pair takes several items)]}, which
as scao_gated_ff_plan has it (0 the forward pass, 1 dx, 2 dW, 3 both)."""
import ctypes

from scao_b200 import _lib

SINGLE, PAIR, TALL = range(3)
PATHS = {
    (2317, 1761, 4591): [(0, PAIR, 1, 1, True), (2, TALL, 1, 1, True), (3, TALL, 1, 1, True)],
    (4096, 2048, 8192): [(0, TALL, 1, 1, True), (1, TALL, 1, 1, False), (2, PAIR, 1, 1, True), (3, TALL, 1, 1, True)],
    (9000, 300, 2000): [(0, TALL, 1, 1, True), (2, PAIR, 1, 2, False), (3, PAIR, 1, 1, True)],
    (2549, 173, 1214): [(0, SINGLE, 1, 1, True), (1, SINGLE, 3, 1, False), (3, PAIR, 3, 3, False)],
    (3381, 248, 3191): [(0, PAIR, 1, 1, True), (1, PAIR, 5, 1, False), (3, PAIR, 2, 1, False)],
    (1531, 1000, 2731): [(0, TALL, 1, 1, False), (1, PAIR, 3, 1, False), (3, PAIR, 2, 1, True)],
    (20000, 300, 1000): [(2, SINGLE, 1, 3, False), (3, PAIR, 1, 4, True)],
}


def plan(rows, d, ff, which):
    """(tile, cuts of dx, cuts of dW, whether a CTA or pair takes several items)."""
    out = (ctypes.c_int32 * 5)()
    assert _lib.lib().scao_gated_ff_plan(rows, d, ff, which, out) == 0
    tile, items, dx, dw, groups = out
    return tile, dx, dw, items > groups
