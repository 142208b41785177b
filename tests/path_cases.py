"""Sizes of the MXFP4 and gated-block calls, with the kernels that each is there for. tests/test_paths.py holds the kernels to
that on the host; tests/test_gpu_mxfp4_paths.py and tests/test_gpu_ffn_paths.py run the calls."""

# M, N, K of products whose scales are read in their stored order, K a multiple of 256 and of 128 alone, and the others
PRODUCTS = [
    (500, 4000, 256, ["mx_matmul_kernel<128,64,2,2,4,0>"]),
    (500, 4000, 384, ["mx_matmul_kernel<128,64,2,2,4,0>"]),
    (60, 70000, 384, ["mx_matmul_kernel<128,64,2,2,4,0>"]),
    (1100, 2000, 512, ["mx_matmul_kernel<128,128,2,2,4,0>"]),
    (1100, 2000, 640, ["mx_matmul_kernel<128,128,2,2,4,0>"]),
    (2100, 2500, 512, ["mx_matmul_kernel<128,128,2,2,2,0>"]),
    (2100, 2500, 640, ["mx_matmul_kernel<128,128,2,2,2,0>"]),
    (100, 66000, 128, ["mx_matmul_kernel<128,128,2,2,2,0>"]),
    (100, 70, 8448, ["mx_matmul_kernel<64,64,2,2,4,0>", "join_kernel"]),
    (100, 70, 16512, ["mx_matmul_kernel<64,64,2,2,4,0>", "join_kernel"]),
    (300, 1900, 8320, ["mx_matmul_kernel<64,64,2,2,4,0>"]),
    (100, 70, 8064, ["mx_matmul_kernel<64,64,2,2,4,1>", "join_kernel"]),
    (100, 70, 384, ["mx_matmul_kernel<64,64,2,2,4,1>"]),
    (4100, 3400, 384, ["mx_arrange_kernel", "mx_matmul_kernel<256,256,2,4,2,0>"]),
    (7, 70, 384, ["mx_matmul_few_kernel<1,1>"]),
    (16, 70, 640, ["mx_matmul_few_kernel<1,2>"]),
    (3, 50, 1152, ["mx_matmul_few_kernel<1,4>"]),
    (33, 70, 2176, ["mx_matmul_few_kernel<1,8>"]),
]

FEW, TILE, WIDE = "mx_gateup_few_kernel<4>", "mx_gateup_kernel<128,64,2,2,3>", "mx_gateup_kernel<128,128,2,2,2>"
DOWN_TILE, DOWN_WIDE = "mx_down_kernel<128,64,2,2,3>", "mx_down_kernel<128,128,2,2,2>"
DIRECT = ["mx_gateup_direct_kernel<2,4>", "mx_down_direct_kernel"]

# experts, hidden, intermediate, tokens, picks, limit, the kernels among the call's: with local ids, and with a map of two more ids than experts
ROUTED = [
    (56, 544, 288, 56, 8, 10.0, [FEW, "mx_down_few_kernel<2,1>"]),
    (40, 192, 1056, 40, 8, 1.0, [FEW, "mx_down_few_kernel<2,4>"]),
    (40, 288, 736, 40, 8, 2.0, [FEW, "mx_down_few_kernel<2,2>"]),
    (40, 96, 2208, 40, 8, 0.0, [FEW, "mx_down_few_kernel<2,8>"]),
    (640, 32, 32, 600, 8, 2.0, [FEW, "mx_down_few_kernel<2,1>"]),
    (16, 544, 288, 120, 4, 10.0, [TILE, DOWN_TILE]),
    (13, 1120, 160, 150, 3, 1.0, [TILE, DOWN_TILE]),
    (64, 64, 96, 700, 6, 2.0, [TILE, DOWN_TILE]),
    (3, 544, 288, 333, 2, 10.0, [WIDE, DOWN_WIDE]),
    (2, 160, 1120, 700, 1, 0.0, [WIDE, DOWN_WIDE]),
    (5, 96, 32, 2100, 2, 2.0, [WIDE, DOWN_WIDE]),
    (3, 16384, 64, 263, 2, 10.0, [WIDE, DOWN_WIDE]),
    (3, 64, 16384, 263, 2, 1.0, [WIDE, DOWN_WIDE]),
    (16, 544, 288, 20, 4, 10.0, DIRECT),
    (9, 16384, 32, 5, 2, 2.0, DIRECT),
]
# the same with hidden and intermediate that are multiples of 128 but not of 256: scales as they come
STORED = [
    (56, 640, 384, 56, 8, [FEW, "mx_down_few_kernel<2,1>"]),
    (16, 640, 384, 120, 4, [TILE, DOWN_TILE]),
    (3, 640, 384, 260, 2, [WIDE, DOWN_WIDE]),
    (16, 640, 384, 20, 4, DIRECT),
]

# tokens, hidden, intermediate, limit, the kernels of the forward pass (bf16; fp16's are the same ones)
FORWARD = [
    (1, 136, 72, 10.0, ["gated_few_kernel<2>"]),
    (40, 264, 136, 1.0, ["gated_few_kernel<2>"]),
    (97, 4168, 1032, 2.0, ["gemm16_kernel<2,0,0,64,64,2,2,4>", "gated_join_kernel<2>"]),
    (130, 264, 776, 10.0, ["gated_kernel<2,128,64,2,2,4>"]),
    (1300, 1096, 1032, 1.0, ["gated_kernel<2,128,128,2,4,4>"]),
    (2050, 136, 2056, 2.0, ["gated_kernel<2,128,128,2,2,2>"]),
    (3339, 392, 2056, 0.0, ["gated_kernel<2,256,256,2,4,2>"]),
]
# the products of the gradients: dx, then dw13
DX = [
    (130, 264, 136, 10.0, ["gemm16_kernel<2,1,0,64,64,2,2,4>"]),
    (130, 264, 2056, 2.0, ["gemm16_kernel<2,1,0,64,64,2,2,4>", "join_kernel"]),
    (1300, 1096, 264, 1.0, ["gemm16_kernel<2,1,0,128,128,2,4,4>"]),
    (2100, 2056, 72, 0.0, ["gemm16_kernel<2,1,0,128,128,2,2,2>"]),
    (3339, 4104, 136, 10.0, ["gemm16_kernel<2,1,0,256,256,2,4,2>"]),
]
DW = [
    (130, 264, 136, 10.0, ["gemm16_kernel<2,1,1,64,64,2,2,4>"]),
    (8203, 136, 72, 2.0, ["gemm16_kernel<2,1,1,64,64,2,2,4>", "join_kernel"]),
    (70, 520, 1032, 1.0, ["gemm16_kernel<2,1,1,128,128,2,4,4>"]),
    (43, 1096, 2056, 0.0, ["gemm16_kernel<2,1,1,128,128,2,2,2>"]),
    (43, 4104, 2056, 10.0, ["gemm16_kernel<2,1,1,256,256,2,4,2>"]),
]
