"""Sizes of the 8-bit tensors' tests by the kernel they are meant for (test_packed8_choice.py holds them to it on the CPU), beside
those of test_packed8_gpu.py. A kernel is named as tests/host/packed8_choice_main.cpp names it, with "split" where k (the rows) is
taken in several parts: ("tile", 0) to ("tile", 5) are k_gemm8<256, 256>, <128, 128>, <128, 64>, <64, 64>, k_gemm8_few<4> and <8>;
("thin", 8, 2) is k_gemm8_thin<8, 2>; ("dw", 0) to ("dw", 3) are k_dw8<4, 2>, <2, 2>, <1, 3> and k_dw8_few<8>."""

CUS = 256  # of an MI355X

# m, n, k
PRODUCTS = [((429, 4749, 11581), ("tile", 0, "split")), ((1, 2769, 19408), ("tile", 4, "split")),
            ((1379, 1, 42508), ("tile", 4, "split")), ((16, 4200, 2000), ("thin", 4, 1)), ((32, 5000, 1300), ("thin", 4, 2)),
            ((48, 4500, 1300), ("thin", 4, 3))]

# A product of each kernel, in one part and in several, for values that are not finite
SPECIAL_PRODUCTS = [((16, 4200, 300), ("thin", 4, 1)), ((32, 5000, 200), ("thin", 4, 2)), ((48, 4500, 700), ("thin", 4, 3)),
                    ((8, 70, 1029), ("thin", 8, 1)), ((17, 33, 640), ("thin", 8, 2)), ((40, 100, 2000), ("thin", 8, 3)),
                    ((4093, 4093, 520), ("tile", 0)), ((1537, 2050, 1300), ("tile", 1)), ((6001, 2050, 300), ("tile", 2)),
                    ((700, 900, 300), ("tile", 3)), ((777, 333, 1000), ("tile", 4)), ((300, 260, 1100), ("tile", 5)),
                    ((429, 4749, 11581), ("tile", 0, "split")), ((777, 1000, 9000), ("tile", 1, "split")),
                    ((4099, 33, 16500), ("tile", 2, "split")), ((260, 1000, 9000), ("tile", 3, "split")),
                    ((1379, 1, 42508), ("tile", 4, "split")), ((130, 260, 9000), ("tile", 5, "split"))]

# rows, in, out: the third kernel with more rows than its ring holds and in several parts, the others with fewer than four columns of g
WEIGHT_GRADIENTS = [((441, 350, 1466), ("dw", 2)), ((521, 69, 5190), ("dw", 2)), ((8571, 15, 685), ("dw", 2, "split")),
                    ((6781, 1, 1418), ("dw", 2, "split")), ((13457, 720, 1), ("dw", 2, "split")), ((698, 101, 4100), ("dw", 0)),
                    ((3672, 3925, 1), ("dw", 0, "split")), ((4746, 1358, 1), ("dw", 1, "split")), ((436, 8382, 1), ("dw", 1))]

# of each kernel, in one part and in several, rows behind the last whole block
SPECIAL_WEIGHT_GRADIENTS = [((698, 101, 4100), ("dw", 0)), ((2600, 1000, 260), ("dw", 0, "split")), ((700, 1000, 333), ("dw", 1)),
                            ((16390, 260, 500), ("dw", 1, "split")), ((521, 69, 5190), ("dw", 2)), ((441, 350, 1466), ("dw", 2)),
                            ((8571, 15, 685), ("dw", 2, "split")), ((300, 77, 40), ("dw", 3)), ((9001, 130, 130), ("dw", 3, "split"))]

# rows, width, hidden of blocks whose weight gradient dw1 and product dw2 leave parts in scratch
SPLIT_BLOCKS = [(5000, 64, 128), (6000, 48, 200)]
