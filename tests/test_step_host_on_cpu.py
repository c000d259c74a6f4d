"""Host side of the step operators, without a GPU: what a list of matrices asks
for, and what the Python entry points do before any kernel is launched."""
from mpi_collectives import step_abi


def matrices(*shapes):
    return (step_abi.Matrix * len(shapes))(*[step_abi.Matrix(4096, 4096, 4096, r, c, 1, 0.1) for r, c in shapes])


def test_small_matrices_need_no_workspace_among_larger_ones():
    """Unless all are precise: then they ride along with the larger ones' products."""
    lib = step_abi.lib()
    mixed, large = matrices((64, 256), (300, 200), (20, 30)), matrices((300, 200))
    assert lib.step_orthogonalize_workspace(mixed, 3, 0) == lib.step_orthogonalize_workspace(large, 1, 0) > 0
    assert lib.step_orthogonalize_workspace(mixed, 3, 1) > lib.step_orthogonalize_workspace(large, 1, 1) > 0
    for precise in (0, 1):
        assert lib.step_orthogonalize_workspace(matrices((64, 256), (20, 30)), 2, precise) == 0
