"""GPU shapes of the adapters' tests whose kernel route is their point, with the route each takes on a 256-CU MI355X
(test_adapter_routes.py checks every label against the built planners on the CPU)."""

CUS = 256

# (M, K, N, K slices, super-steps per unit, form, wrapped): row-split launches. form: "slots" (a slot per unit), "groups"
# (one per group of units), "own" (a wave's whole blocks in registers) or "small" (every unit in flight at once). wrapped: more items (column, lane group) than
# threads, so that a thread takes several, and a last column range so narrow that some thread's first item lies past its
# end and a later one does not.
ROWSPLIT = [
    (5, 512, 152064, 1, 4, "slots", True),     # a vocabulary head
    (8, 640, 152064, 1, 5, "slots", True),
    (5, 3584, 152064, 1, 4, "groups", True),
    (8, 12288, 33856, 4, 4, "slots", True),
    (13, 512, 50304, 1, 4, "slots", True),
    (16, 640, 64000, 1, 5, "slots", True),
    (9, 2560, 65984, 1, 4, "groups", True),    # the drafter's vocabulary, one row in the last lane group
    (13, 1024, 21760, 2, 4, "slots", True),
    (16, 5120, 21760, 2, 4, "slots", True),
    (13, 4096, 32000, 2, 4, "slots", True),
    (16, 5120, 33856, 2, 5, "slots", True),
    (3, 1024, 4096, 1, 4, "slots", False),
    (5, 12288, 21760, 4, 4, "slots", False),   # more items than threads, ranges all whole
    (5, 8192, 17408, 1, 4, "groups", False),
    (6, 1024, 5120, 2, 4, "slots", False),
    (8, 512, 2048, 1, 4, "small", False),
    (9, 12288, 2048, 4, 4, "slots", False),
    (16, 5120, 50304, 4, 5, "slots", False),
    (4, 640, 10240, 1, 5, "slots", False),
    (1, 12288, 5120, 2, 4, "slots", False),
    (1, 6400, 176160, 2, 5, "slots", False),
    (3, 5120, 248320, 1, 4, "groups", False),
    (6, 2560, 7168, 2, 5, "slots", False),
    (9, 512, 589824, 1, 4, "own", False),      # whole blocks to each wave
]

# (M, K, N, form): GEMM launches. Whole 256 x 256 tiles with waves split by role ("whole") or not ("whole, plain": K not a
# multiple of 512), what a last round leaves as 128 x 128 quarters or as stream-K over the quarters, and stream-K over each tile.
GEMM = [
    (2304, 512, 4096, "whole"),
    (2048, 512, 4096, "quarters"),               # half the CUs' whole tiles, all cut
    (2000, 1024, 4112, "whole"),                 # a partial last row and column of tiles
    (2000, 640, 4112, "whole, plain"),
    (5100, 512, 3312, "whole, tail in stream-K"),
    (5100, 512, 4336, "whole, tail in quarters"),
    (5100, 640, 4336, "whole, plain, tail in quarters"),
    (600, 12288, 4112, "stream-K 256x256"),
    (136, 5120, 10256, "stream-K 128x256"),
    (203, 5120, 17408, "stream-K 128x256"),      # in units of 4 K steps
    (515, 2048, 1040, "stream-K 128x128"),
    (129, 2048, 10240, "stream-K 128x128"),      # in units of 4 K steps
    (300, 640, 4112, "stream-K 128x128, plain"),
]

# (M, K, N, variant of the row-phase kernel, K split): 28 variants less those that no shape takes.
ROWPHASE = [
    (33, 1024, 17408, 2, True), (33, 512, 99984, 2, False), (9, 20480, 8192, 3, True), (17, 4096, 17408, 4, True),
    (48, 2048, 17408, 5, True), (12, 20480, 512, 6, True), (24, 1024, 272, 7, True), (17, 512, 256, 7, False),
    (64, 512, 272, 8, True), (33, 512, 17408, 8, False), (9, 20480, 1024, 9, True), (24, 8192, 2064, 10, True),
    (12, 5120, 99984, 11, False), (17, 512, 99984, 12, False), (72, 2048, 17408, 13, True), (65, 512, 272, 14, True),
    (72, 512, 17408, 14, False), (81, 2048, 17408, 15, True), (96, 512, 272, 16, True), (90, 512, 17408, 16, False),
    (100, 2048, 17408, 17, True), (112, 512, 272, 18, True), (97, 512, 17408, 18, False), (120, 512, 272, 19, True),
    (24, 512, 32784, 20, False), (48, 512, 32784, 21, False), (17, 512, 65984, 22, False), (64, 512, 65984, 23, False),
    (65, 512, 32784, 24, False), (90, 512, 32784, 25, False), (9, 5120, 65984, 26, False), (12, 8192, 32784, 27, False),
]

# (M, K, N): what no other kernel takes, up to 64 rows. From 5 rows K that is not a multiple of 512 (the verify kernel),
# up to 4 rows too little work for the row-split kernel (the skinny kernel: K in steps of 1, 2 and 4 x 128).
VERIFY = [(6, 128, 48), (9, 384, 272), (16, 768, 2064), (17, 1152, 528), (32, 1280, 4112), (33, 640, 528), (64, 2432, 5136)]
SKINNY = [(1, 128, 16), (3, 2176, 5120), (4, 256, 5136), (2, 768, 272), (1, 20480, 2048), (3, 20480, 48), (4, 20480, 528)]
