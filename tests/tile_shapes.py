"""Shapes that reach every tile of the batched products of orthogonalised updates and of the
8-bit products (test_tiles_covered.py asks the planner that they do, test_gpu_tiles.py runs them)."""

# batch, rows, cols; each as it is and transposed, with products of two parts and fast ones.
ORTH = [
    (1, 16, 16),
    (3, 40, 70),
    (32, 65, 65),
    (64, 129, 134),
    (16, 16, 258),
    (32, 16, 518),
    (64, 193, 197),
    (32, 65, 1977),
    (64, 66, 784),
    (64, 328, 599),
    (32, 578, 581),
    (16, 579, 593),
    (16, 898, 928),
    (16, 1157, 1175),
    (16, 1177, 1500),
    (8, 1676, 1760),
    (8, 917, 1549),
    (4, 2443, 2446),
    (4, 910, 3094),
    (1, 3244, 3802),
    (32, 66, 970),
    (1, 2048, 2048),
]

# rows, in, out, layout ("odd": rows and their ends lie anywhere)
INT8 = [
    # up to 64 rows kept in LDS: work-groups of one block of columns and of several, waves with
    # columns of their own, and 16-bit results stored in lines
    (2, 100, 9001, "odd"),
    (16, 1300, 70, "dense"),
    (16, 1301, 5000, "odd"),
    (20, 1100, 32801, "odd"),
    (64, 600, 33000, "dense"),
    # as many rows too long for that, and more
    (18, 15, 40, "odd"),
    (9, 15, 17920, "odd"),
    (20, 9000, 70, "dense"),
    (20, 9001, 16600, "odd"),
    (70, 32, 16, "dense"),
    (69, 19, 17, "odd"),
    (68, 16, 8768, "dense"),
    (8952, 3642, 71, "odd"),
    (8615, 16, 66, "odd"),
    (2620, 16, 2856, "dense"),
    (10688, 32, 584, "dense"),
    (7756, 776, 769, "odd"),
    (6431, 656, 464, "dense"),
    (5018, 32, 704, "dense"),
    (9575, 662, 336, "odd"),
    (2963, 21, 1188, "odd"),
    (700, 1537, 8195, "odd"),
    (9877, 2961, 1197, "odd"),
    (5981, 5760, 2112, "dense"),
    # the reduction in parts
    (99, 3136, 16, "dense"),
    (133, 3516, 16, "odd"),
    (4097, 7152, 16, "dense"),
    (2049, 14000, 16, "dense"),
    (1213, 27895, 16, "odd"),
    (3385, 37152, 72, "dense"),
    (10324, 17920, 72, "dense"),
    (3364, 27712, 96, "dense"),
    (3455, 26768, 80, "dense"),
    (613, 62189, 260, "odd"),
    (907, 117758, 112, "odd"),
    (7115, 69485, 149, "odd"),
    (6927, 61104, 136, "dense"),
]
