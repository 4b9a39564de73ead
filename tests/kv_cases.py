"""Calls of attention that take each variant of the kernel for few rows, with sequences that several workgroups share."""

# head size padded to, 16s of rows, waves: lengths of the sequences, rows of each (None: one, without starts), query heads, key/value heads, head size
SHARED = {
    (64, 1, 4): ([300 + 7 * i for i in range(40)], None, 32, 8, 64),
    (64, 1, 8): ([3000, 2100], [2, 3], 16, 4, 40),
    (128, 1, 4): ([3000, 700, 2222], None, 32, 16, 128),
    (128, 1, 8): ([5000, 4100], [2, 1], 16, 4, 96),
    (256, 1, 4): ([3000, 700, 40], [3, 2, 3], 16, 4, 200),
    (64, 2, 4): ([400 + 5 * i for i in range(20)], [20] * 20, 16, 16, 64),
    (64, 2, 8): ([3000, 2500], [20, 17], 16, 16, 64),
    (128, 2, 4): ([9000, 8500], [30, 17], 16, 16, 100),
}
