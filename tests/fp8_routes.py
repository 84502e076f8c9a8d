"""A product for each kernel that multiplies 8-bit rows and weights, and a norm for each of its: sizes, with the kernel that they
take. The sizes are ragged: last tiles that are not whole, columns that are not whole blocks, stretches of k of different lengths."""

# rows of A, rows of B, columns, whether C is f32, kernel, stretches of k
PRODUCTS = [
    (m, n, k, f32, kernel % (2 if m > 8 else 1), 1)
    for n, k, kernel in ((300, 520, "fp8_stream_kernel<%d,1,4,3,1>"), (4201, 600, "fp8_stream_kernel<%d,2,4,3,1>"), (8301, 600, "fp8_stream_kernel<%d,2,4,2,1>"),
                         (8301, 2100, "fp8_stream_kernel<%d,4,4,2,1>"), (301, 4200, "fp8_stream_kernel<%d,1,8,2,1>"), (4300, 8300, "fp8_stream_kernel<%d,1,8,2,1>"))
    for m, f32 in ((1, False), (7, True), (9, False), (15, True))
] + [
    (m, n, k, f32, kernel % f32, 1)
    for m, n, k, kernel in ((18, 301, 600, "fp8_stream_kernel<4,1,4,3,%d>"), (41, 301, 600, "fp8_stream_kernel<6,1,4,2,%d>"), (61, 301, 600, "fp8_stream_kernel<8,1,4,2,%d>"),
                            (31, 4201, 600, "fp8_stream_kernel<4,2,4,3,%d>"), (47, 4201, 600, "fp8_stream_kernel<6,2,4,3,%d>"), (63, 4201, 600, "fp8_stream_kernel<8,2,4,2,%d>"),
                            (20, 8192, 600, "fp8_stream_kernel<4,2,4,3,%d>"), (64, 8192, 520, "fp8_stream_kernel<8,2,4,2,%d>"),
                            (20, 8300, 600, "fp8_tile_kernel<64,64,2,2,4,%d,1>"), (61, 8301, 600, "fp8_tile_kernel<64,64,2,2,4,%d,1>"))
    for f32 in (False, True)
] + [
    (40, 132, 12400, False, "fp8_tile_kernel<64,64,2,2,4,0,1>", 8),
    (50, 1001, 12400, False, "fp8_tile_kernel<64,64,2,2,4,0,1>", 8),
    (50, 1001, 12400, True, "fp8_tile_kernel<64,64,2,2,4,1,1>", 8),
    (40, 4200, 12400, False, "fp8_tile_kernel<64,64,2,2,4,0,1>", 4),
    (65, 130, 600, False, "fp8_tile_kernel<64,64,2,2,4,0,0>", 1),
    (70, 389, 2100, False, "fp8_tile_kernel<64,64,2,2,4,0,0>", 4),
    (99, 128, 4200, False, "fp8_tile_kernel<64,64,2,2,4,0,0>", 8),
    (65, 130, 600, True, "fp8_tile_kernel<64,64,2,2,4,1,0>", 1),
    (70, 389, 2100, True, "fp8_tile_kernel<64,64,2,2,4,1,0>", 4),
    (99, 128, 4200, True, "fp8_tile_kernel<64,64,2,2,4,1,0>", 8),
    (2049, 1001, 600, False, "fp8_tile_kernel<128,128,4,2,3,0,0>", 1),
    (129, 3001, 8200, False, "fp8_tile_kernel<128,128,4,2,3,0,0>", 4),
    (65, 2100, 8200, False, "fp8_tile_kernel<128,128,4,2,3,0,0>", 8),
    (2049, 1001, 600, True, "fp8_tile_kernel<128,128,4,2,3,1,0>", 1),
    (129, 3001, 8200, True, "fp8_tile_kernel<128,128,4,2,3,1,0>", 4),
    (333, 11201, 600, False, "fp8_tile_kernel<192,128,4,2,3,0,0>", 1),
    (1300, 3008, 600, False, "fp8_tile_kernel<192,128,4,2,3,0,0>", 1),
    (333, 3001, 8200, False, "fp8_tile_kernel<192,128,4,2,3,0,0>", 4),
    (2000, 3001, 600, False, "fp8_tile_kernel<128,128,2,2,2,0,0>", 1),
    (1301, 2999, 600, True, "fp8_tile_kernel<128,128,2,2,2,1,0>", 1),
    (65, 8301, 8200, True, "fp8_tile_kernel<128,128,2,2,2,1,0>", 4),
    (2001, 4101, 600, False, "fp8_tile_kernel<256,256,4,2,2,0,0>", 1),
    (1801, 4504, 1000, False, "fp8_tile_kernel<256,256,4,2,2,0,0>", 1),
]

# columns, kernel
NORMS = [(1, "fp8_norm_kernel<1>"), (2048, "fp8_norm_kernel<1>"), (2049, "fp8_norm_kernel<2>"), (4096, "fp8_norm_kernel<2>"), (4097, "fp8_norm_kernel<4>"),
         (5001, "fp8_norm_kernel<4>"), (5120, "fp8_norm_kernel<4>"), (8192, "fp8_norm_kernel<4>"), (8193, "fp8_norm_kernel<0>")]
