"""Sizes that reach each kernel form of the linear layer, with ragged ends: what
tests/test_layers_plan.py asserts of the choice (layers_plan.h) and
tests/test_gpu_layers_forms.py runs."""

# (form, 16-column tiles or P tile, 16-row tiles or Q tile, splits) -> sizes of a product
# [rows, nc] x [ni, nc]^T: (rows, ni, nc). Splits: 1, or 2 for "several, the last one short".
BF16 = {
    ("fused", 1, 1, 1): (5, 130, 257),
    ("fused", 2, 1, 1): (11, 8190, 150),
    ("fused", 1, 2, 1): (29, 1000, 333),
    ("fused", 2, 2, 1): (20, 8187, 257),
    ("fused", 1, 4, 1): (61, 70, 500),
    ("stream", 1, 4, 1): (60, 900, 4001),
    ("stream", 2, 4, 1): (55, 8190, 1150),
    ("tiles", 64, 64, 1): (131, 200, 333),
    ("tiles", 64, 64, 2): (97, 33, 2050),
    ("tiles", 128, 64, 1): (1001, 1500, 1111),
    ("tiles", 128, 64, 2): (65, 1030, 6000),
    ("tiles", 128, 128, 1): (1300, 2050, 2050),
    ("tiles", 128, 128, 2): (66, 2050, 5900),
    ("tiles", 256, 128, 1): (1030, 4001, 300),
    ("tiles", 256, 128, 2): (193, 4200, 4200),
    ("tiles", 256, 256, 1): (2049, 4001, 260),
    ("tiles", 256, 256, 2): (134, 5891, 10808),
}
# fp32 activations: four tiles of rows are never quantised on the way
F32 = {
    ("fused", 1, 1, 1): (5, 130, 257),
    ("fused", 2, 1, 1): (11, 8190, 150),
    ("fused", 1, 2, 1): (29, 1000, 333),
    ("fused", 2, 2, 1): (20, 8187, 257),
    ("stream", 1, 4, 1): (61, 70, 500),
    ("stream", 2, 4, 1): (60, 8190, 150),
    ("tiles", 128, 64, 1): (1001, 1500, 1111),
}

# (columns of x, of dy, splits as above) -> (rows, n, k) of a weight gradient; odd sizes go
# through copies of the operands, even ones are read in place
OUTER = {
    (128, 128, 1): [(333, 300, 190), (333, 301, 189)],
    (128, 128, 2): [(2049, 130, 250), (2049, 129, 251)],
    (128, 256, 1): [(65, 1030, 4002), (66, 1031, 4001)],
    (128, 256, 2): [(3000, 4200, 6), (3000, 4201, 5)],
    (256, 256, 1): [(70, 2050, 6000), (66, 2051, 5999)],
    (256, 256, 2): [(4700, 14, 4146), (4700, 13, 4147)],
}

# (rows, n, k) of a backward pass whose dx would take tiles of 128 x 64 and runs in 64 x 64
# beside dw, and of passes that do not run in one launch
BACKWARD_IN_ONE = [(1001, 1500, 1111), (1001, 1500, 1112)]
BACKWARD_APART = [(1300, 2050, 2050), (130, 4001, 300), (2049, 260, 4001)]
