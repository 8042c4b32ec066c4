"""Sizes that together take every tile shape of every product of the hidden-state
operators (test_head_plan.py says which; test_gpu_head_large.py runs them).  None
is a multiple of a tile, so that every shape has ragged last tiles."""

# dtype "16": bfloat16 and float16 in turn; operator, dtype, rows, in (hidden), out
# (vocabulary), layout
SHAPES = [
    ("linear", "16", 87, 40, 8208, "pad"),
    ("linear", "16", 84, 21, 8856, "pad"),
    ("linear", "16", 7298, 72, 968, "dense"),
    ("linear", "16", 1834, 20, 4024, "dense"),
    ("linear", "16", 6210, 264, 456, "dense"),
    ("linear", "16", 3895, 712, 3344, "pad"),
    ("linear", "16", 74, 1864, 75, "pad"),
    ("linear", "16", 66, 1793, 89, "odd"),
    ("linear", "16", 8979, 4747, 66, "odd"),
    ("linear", "16", 231, 4792, 4225, "pad"),
    ("linear", "f32", 84, 447, 69, "dense"),
    ("linear", "f32", 82, 440, 72, "pad"),
    ("linear", "f32", 8822, 16, 83, "dense"),
    ("linear", "f32", 8426, 20, 114, "odd"),
    ("linear", "f32", 2858, 34, 1104, "odd"),
    ("linear", "f32", 1445, 36, 2200, "dense"),
    ("linear", "f32", 7023, 16, 1064, "pad"),
    ("linear", "f32", 69, 4552, 528, "dense"),
    ("linear", "f32", 72, 4669, 593, "odd"),
    ("linear", "f32", 8380, 2792, 80, "dense"),
    ("linear_backward", "16", 8855, 80, 72, "pad"),
    ("linear_backward", "16", 70, 142, 5700, "odd"),
    ("linear_backward", "16", 3271, 284, 65, "odd"),
    ("linear_backward", "16", 65, 216, 4307, "pad"),
    ("linear_backward", "16", 65, 4264, 1456, "dense"),
    ("linear_backward", "16", 2177, 2875, 66, "odd"),
    ("linear_backward", "16", 5052, 20, 6053, "odd"),
    ("linear_backward", "16", 73, 2386, 5627, "odd"),
    ("linear_backward", "16", 8804, 2054, 71, "odd"),
    ("linear_backward", "16", 881, 3632, 981, "dense"),
    ("linear_backward", "16", 6863, 2096, 728, "dense"),
    ("linear_backward", "16", 6980, 1864, 825, "odd"),
    ("linear_backward", "16", 600, 2563, 7200, "dense"),
    ("linear_backward", "16", 913, 1688, 8024, "pad"),
    ("linear_backward", "f32", 500, 16, 416, "pad"),
    ("linear_backward", "f32", 433, 25, 518, "odd"),
    ("linear_backward", "f32", 5067, 16, 1194, "dense"),
    ("linear_backward", "f32", 67, 271, 7751, "odd"),
    ("linear_backward", "f32", 67, 304, 7728, "dense"),
    ("linear_backward", "f32", 2588, 1068, 66, "odd"),
    ("linear_backward", "f32", 4809, 552, 80, "pad"),
    ("linear_backward", "f32", 1162, 4432, 72, "pad"),
    ("linear_backward", "f32", 465, 4200, 488, "dense"),
    ("linear_backward", "f32", 456, 4456, 481, "odd"),
    ("linear_backward", "f32", 74, 4512, 6358, "dense"),
    ("linear_backward", "f32", 6041, 66, 5752, "dense"),
    ("head", "16", 87, 16, 8208, "pad"),
    ("head", "16", 7298, 16, 968, "dense"),
    ("head", "16", 6210, 264, 456, "dense"),
    ("head", "16", 4972, 726, 2544, "dense"),
    ("head", "16", 8855, 80, 72, "pad"),
    ("head", "16", 70, 142, 5700, "odd"),
    ("head", "16", 266, 3370, 67, "odd"),
    ("head", "16", 65, 216, 4307, "pad"),
    ("head", "16", 2177, 2875, 66, "odd"),
    ("head", "16", 8759, 22, 2760, "dense"),
    ("head", "16", 73, 2386, 5627, "odd"),
    ("head", "16", 352, 880, 8808, "pad"),
    ("head", "16", 846, 3758, 909, "dense"),
    ("head", "16", 6863, 2096, 728, "dense"),
    ("head", "16", 391, 4888, 6922, "odd"),
    ("head", "16", 1448, 1656, 8544, "dense"),
    ("head", "f32", 8822, 16, 83, "dense"),
    ("head", "f32", 7146, 16, 408, "pad"),
    ("head", "f32", 967, 16, 7034, "dense"),
    ("head", "f32", 433, 25, 518, "odd"),
    ("head", "f32", 653, 16, 1499, "dense"),
    ("head", "f32", 5114, 16, 1375, "pad"),
    ("head", "f32", 67, 271, 7751, "odd"),
    ("head", "f32", 193, 4664, 200, "dense"),
    ("head", "f32", 1211, 76, 2659, "odd"),
    ("head", "f32", 446, 4795, 152, "odd"),
    ("head", "f32", 195, 4157, 641, "odd"),
    ("head", "f32", 465, 4200, 488, "dense"),
    ("head", "f32", 6531, 4296, 65, "odd"),
    ("head", "f32", 74, 4512, 6358, "dense"),
]

# rows, hidden, vocabulary of bfloat16 heads whose last piece is 1, 2, 3 and 4 slabs
# of the reduction of d_x on the 256 x 256 tile, added to the pieces before it
LAST_PIECES = [(18000, 1544, 46593), (18000, 1544, 46662), (18000, 1544, 46742), (18000, 1544, 46842)]

# rows, hidden, vocabulary, layout of heads in several pieces whose weight is copied
# piece by piece, in both directions
COPIED = [("16", 1290, 4099, 37003, "odd"), ("f32", 1290, 2051, 37003, "odd")]

# dtype, rows, in, out of linear blocks whose output and pre-activations are stored
# past the caches
STREAMED = [("bf16", 4500, 4104, 6330), ("f16", 4500, 4104, 6330), ("f32", 4110, 72, 4100)]
