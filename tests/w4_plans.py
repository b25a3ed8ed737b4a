"""Shapes of 4-bit products and the launches that they take: what tests/test_gpu_w4_plans.py runs, and
tests/test_w4_plans.py holds against the rules, so that a rule that changes cannot leave a kernel without a test."""
import ctypes as C

FEW, STREAM, BATCH, TILE = range(4)

# (tokens, rows, columns) -> (kernel, tiles of a wave or 64s of tokens, waves, spans of k, steps of 128 k in a span).
PLANS = {
    # Few tokens.
    (1, 16, 128): (FEW, 1, 16, 1, 1), (9, 300, 4096): (FEW, 1, 16, 1, 32), (4, 3000, 8192): (FEW, 1, 16, 1, 64),
    (2, 8193, 1152): (FEW, 2, 16, 1, 9), (9, 5000, 4096): (FEW, 2, 16, 1, 32), (16, 20000, 640): (FEW, 4, 16, 1, 5),
    # Streams: all of x in LDS, and in chunks.
    (4, 32768, 6912): (STREAM, 2, 8, 1, 54), (4, 32769, 7168): (STREAM, 2, 8, 1, 56), (1, 32771, 28672): (STREAM, 2, 8, 1, 224),
    # Batches of four waves, up to 16, 32 and 64 tokens: spans of more than 32 steps in one piece and in spans.
    (16, 32710, 4352): (BATCH, 1, 4, 1, 34), (17, 32711, 4480): (BATCH, 1, 4, 1, 36), (64, 32712, 4352): (BATCH, 1, 4, 1, 34),
    (16, 300, 67072): (BATCH, 1, 4, 16, 34), (24, 300, 67200): (BATCH, 1, 4, 16, 34), (61, 300, 67072): (BATCH, 1, 4, 16, 34),
    # Sixteen waves, up to 16 tokens, and up to 32 with two tiles a wave; eight, up to 64.
    (7, 90113, 4480): (BATCH, 1, 16, 1, 36), (16, 33000, 4096): (BATCH, 1, 16, 3, 12), (16, 32769, 12928): (BATCH, 1, 16, 3, 34),
    (19, 262145, 4352): (BATCH, 2, 16, 1, 34), (20, 33001, 2816): (BATCH, 2, 16, 4, 6), (32, 33000, 34944): (BATCH, 2, 16, 8, 36),
    (64, 65537, 4480): (BATCH, 1, 8, 1, 36), (64, 32769, 2816): (BATCH, 1, 8, 2, 12), (40, 32770, 4224): (BATCH, 1, 8, 2, 18),
    (33, 32769, 8832): (BATCH, 1, 8, 2, 36),
    # Tiles of 64 and of 128 tokens; their loop ends after 0, 2 or 4 of six chunks of 64 k.
    (100, 257, 128): (TILE, 1, 4, 1, 1), (513, 2816, 640): (TILE, 1, 4, 1, 5), (127, 96, 896): (TILE, 1, 4, 1, 7), (1000, 1111, 768): (TILE, 1, 4, 1, 6),
    (300, 400, 4096): (TILE, 1, 4, 8, 4), (255, 63, 2816): (TILE, 1, 4, 5, 5), (129, 129, 1536): (TILE, 1, 4, 3, 4), (90, 16, 65536): (TILE, 1, 4, 16, 32),
    (2050, 1111, 128): (TILE, 2, 4, 1, 1), (4099, 401, 256): (TILE, 2, 4, 1, 2), (4099, 401, 768): (TILE, 2, 4, 1, 6), (300, 8192, 896): (TILE, 2, 4, 1, 7),
    (500, 5001, 640): (TILE, 2, 4, 1, 5), (65, 2816, 4096): (TILE, 2, 4, 8, 4), (700, 130, 8192): (TILE, 2, 4, 16, 4), (4099, 16, 2816): (TILE, 2, 4, 5, 5),
    (16384, 17, 2816): (TILE, 2, 4, 2, 11),
}


def plan(tokens, rows, cols):
    from inferno_amd._lib import I64, P_I64, lib

    fn = lib().ifr_internal_w4_plan
    fn.restype, fn.argtypes = C.c_int32, [I64, I64, I64, P_I64]
    out = (C.c_int64 * 5)()
    return tuple(out) if fn(rows, cols, tokens, out) == 0 else None
