"""Sizes of products with an epilogue by the kernel that the sizes' rule gives them: rows by
weight rows of a tile and slices of K, with and without SwiGLU.  ``test_experts_calls`` holds the
rule to them and ``test_gpu_experts_paths`` runs them."""

from __future__ import annotations

# (rows, weight rows): of a size's last tile of rows one to all of its 16-row blocks are filled; odd columns, and
# columns that end with a tile; more than eight tiles of rows, which go through the columns in bands
WHOLE = {
    (64, 32): {None: [(5, 9, 72), (31, 130, 520), (70, 64, 200), (531, 33, 72)],
               "swiglu": [(5, 9, 72), (33, 64, 520), (545, 65, 200)]},
    (64, 128): {None: [(5, 8199, 200), (17, 8256, 520), (33, 8207, 200), (2339, 197, 520), (594, 832, 200)],
                "swiglu": [(5, 4160, 200), (17, 4129, 200), (33, 4137, 520), (2319, 97, 520), (801, 320, 200)]},
    (128, 256): {None: [(129, 10973, 200), (162, 11200, 200), (195, 8227, 640), (2375, 775, 520), (1601, 1216, 200)],
                 "swiglu": [(129, 5583, 200), (161, 5504, 640), (66, 8367, 520), (1604, 583, 640), (1218, 832, 200)]},
    (256, 256): {None: [(517, 13267, 200), (546, 13120, 200), (585, 13211, 520), (643, 10944, 640), (2306, 3329, 520)],
                 "swiglu": [(258, 11005, 200), (292, 10944, 640), (322, 10885, 520), (385, 8384, 640), (2305, 1691, 520)]},
}

# and slices of K
SLICED = {
    (64, 32, 2): {None: (5, 1645, 6072), "swiglu": (5, 836, 5928)},
    (64, 32, 4): {None: (5, 8, 3800), "swiglu": (5, 8, 3800)},
    (64, 128, 2): {None: (5, 5376, 8288), "swiglu": (5, 3253, 6744)},
    (64, 128, 4): {None: (3202, 8, 6008), "swiglu": (5, 1896, 11616)},
    (128, 256, 2): {None: (136, 11027, 2048), "swiglu": (77, 8377, 1928)},
    (128, 256, 4): {None: (65, 8464, 4112), "swiglu": (71, 4285, 3864)},
    (128, 256, 8): {None: (18, 2727, 10688), "swiglu": (22, 1374, 9728)},
    (256, 256, 2): {None: (262, 13081, 4208), "swiglu": (67, 8474, 2120)},
    (256, 256, 4): {None: (5, 6351, 7784), "swiglu": (5, 3050, 7200)},
    (256, 256, 8): {None: (18, 2733, 10112), "swiglu": (17, 1310, 9024)},
}

SIZES = ([(M, N, K, act, (*tile, 1)) for tile, acts in WHOLE.items() for act, sizes in acts.items() for M, N, K in sizes]
         + [(*size, act, tile) for tile, acts in SLICED.items() for act, size in acts.items()])
