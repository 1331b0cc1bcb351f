"""CPU-only checks of what the entry points around a linear layer ask a caller for, and of the sizes that they take."""
import fbcuda_amd as F


def test_matrices_that_stay_on_chip_want_no_more_workspace_in_batches():
    size = F.orthogonalize_workspace
    for rows, cols in ((1, 1), (2, 3), (64, 64), (64, 300), (96, 192), (192, 96), (64, 480), (32, 1152)):
        one = size(1, rows, cols)
        assert 512 < one < 1 << 20
        for batch in (2, 65536, (1 << 22) - 1, 1 << 22, 1 << 24):
            assert size(batch, rows, cols) == one
    for rows, cols in ((97, 97), (64, 481), (500, 500)):  # these lie in it
        assert size(2, rows, cols) > size(1, rows, cols) > 8 * rows * cols
