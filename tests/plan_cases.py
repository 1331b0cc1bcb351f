"""Sizes for which each kernel of the products around a linear layer is the one that runs on 256 compute units, most of them ragged:
the GPU tests run them, and a test without a GPU holds them against the plans themselves."""

# (M, K, N), whether x comes as codes (or its columns apart), and the plan: way (x quantised by the workgroups) or few, with their
# blocks of 16 rows of x and of w; or tiles, with their side, the ranges of k, and the blocks of 32 k in a range
MX4 = [
    ((3, 100, 30), False, "way 1 1"), ((11, 70, 5003), False, "way 1 2"), ((3, 100, 30), True, "few 1 1"), ((9, 70, 5003), True, "few 1 2"),
    ((4273, 40, 9), True, "few 2 1"), ((437, 3297, 333), False, "few 2 1"), ((135, 86, 997), True, "few 2 2"), ((684, 1318, 333), False, "few 2 2"),
    ((1030, 90, 1531), True, "few 4 1"), ((5518, 373, 102), False, "few 4 1"), ((33, 45, 4071), True, "few 4 2"), ((609, 456, 712), False, "few 4 2"),
    # tiles in one range: fewer blocks than a step has, some more than whole steps, whole steps
    ((2500, 100, 3001), False, "tiles 128 1 8"), ((3000, 200, 1531), True, "tiles 128 1 8"), ((978, 417, 849), True, "tiles 128 1 16"),
    ((1111, 1151, 1009), False, "tiles 128 1 40"), ((1025, 520, 1031), True, "tiles 128 1 24"), ((1280, 512, 1024), False, "tiles 128 1 16"),
    ((3000, 60, 3001), False, "tiles 256 1 8"), ((1031, 333, 7183), True, "tiles 256 1 16"), ((1027, 2100, 7201), False, "tiles 256 1 72"),
    ((2048, 512, 8192), False, "tiles 256 1 16"),
    # in several, joined a result to a lane, to eight lanes, and in words
    ((260, 4352, 1300), False, "tiles 128 6 24"), ((75, 9940, 67), True, "tiles 128 20 16"), ((264, 4352, 1304), False, "tiles 128 6 24"),
    ((512, 4096, 1024), False, "tiles 128 4 32"), ((2156, 15582, 142), False, "tiles 256 16 32"),
]

# (matrices, rows, columns), and the plans of X X^T, A A and B X: kernel, side of its tiles, ranges of k, and k in a range
PAIRS = [
    ((1, 98, 97), "small16 16 1 128 small16 16 1 128 small16 16 1 128"),
    ((7, 99, 100), "small16 16 1 128 small16 16 1 128 small32 32 1 128"),
    ((13, 98, 106), "small32 32 1 128 small32 32 1 128 small32 32 1 128"),
    ((1, 90, 1509), "small32 32 6 256 small16 16 1 96 small32 32 1 96"),
    ((27, 113, 97), "deep64 64 1 128 deep64 64 1 128 deep64 64 1 128"),
    ((3, 97, 2164), "deep64 64 8 288 small16 16 1 128 deep64 64 1 128"),
    ((44, 402, 136), "wide64 64 1 416 deep64 64 1 160 deep64 64 1 160"),
    ((58, 134, 136), "deep64 64 1 160 deep64 64 1 160 wide64 64 1 160"),
    ((58, 205, 198), "wide64 64 1 224 wide64 64 1 224 wide128 128 1 224"),
    ((33, 90, 4211), "wide64 64 4 1056 small32 32 1 96 wide128 128 1 96"),
    ((4, 1483, 389), "deep64 64 1 1504 deep64 64 1 416 deep128 128 1 416"),
    ((64, 193, 598), "deep128 128 1 608 deep64 64 1 224 wide128 128 1 224"),
    ((31, 3203, 206), "deep128 128 2 1632 deep64 64 1 224 wide128 128 1 224"),
    ((19, 507, 452), "deep128 128 1 512 deep128 128 1 480 deep64 64 1 480"),
    ((37, 391, 329), "wide128 128 1 416 wide128 128 1 352 wide128 128 1 352"),
    ((13, 321, 2730), "wide128 128 3 928 deep64 64 1 352 wide128 128 1 352"),
    ((1, 1000, 8000), "wide128 128 6 1344 deep64 64 1 1024 wide128 128 1 1024"),
    ((1, 2047, 8000), "wide128 128 3 2688 wide64 64 1 2048 wide256 256 1 2048"),
    ((1, 8000, 2047), "wide128 128 3 2688 wide64 64 1 2048 wide256 256 1 2048"),
    ((56, 133, 8075), "wide64 64 2 4064 deep64 64 1 160 wide256 256 1 160"),
    ((59, 1464, 455), "wide256 256 1 1472 deep64 64 1 480 wide128 128 1 480"),
    ((8, 1412, 1469), "wide256 256 1 1472 wide256 256 1 1440 wide128 128 1 1440"),
    ((1, 3406, 3202), "wide256 256 2 1728 wide128 128 2 1632 wide256 256 1 3232"),
]
