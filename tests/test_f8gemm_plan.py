"""The 8-bit product's kernel choice, computed on the host, over grids of sizes: every answer is a kernel that takes the operands."""
import itertools

import pytest

from backup_1_amd import capi

SIZES = (1, 2, 15, 16, 17, 64, 65, 127, 128, 129, 500, 1000, 2048, 4096, 8192, 20000)


@pytest.mark.parametrize("type_", (capi.F32, capi.F16, capi.BF16))
@pytest.mark.parametrize("scale", (capi.SCALE_F32, capi.SCALE_E8M0))
@pytest.mark.parametrize("b_rows", (1, 128))
def test_choice_fits_the_operands(type_, scale, b_rows):
    plan = capi.lib().decx_hip_f8gemm_plan
    for M, N, K in itertools.product(SIZES, SIZES, (1, 128, 1500, 8192)):
        up = -(-K // 16) * 16
        assert plan(M, N, K, type_, scale, b_rows, up + 1, up, 1) in (1, 2, 3, 4)         # a pitch off the 16-byte grid
        assert plan(M, N, K, type_, scale, b_rows, up, up, 0) in (1, 2, 3, 4)             # a pointer off it
        assert plan(M, N, K, type_, scale, b_rows, 1 << 24, up, 1) in (1, 2, 3, 4)        # 256 rows of it pass 32 bits
        got = plan(M, N, K, type_, scale, b_rows, up, up, 1)
        assert got in (1, 2, 3, 4, 5, 6)
        if got == 6:
            assert type_ != capi.F32 and (scale == capi.SCALE_E8M0 or b_rows == 128)
        if M <= 16 and K >= 1500:
            assert got in (1, 2, 3, 4)                                              # a token's rows fill no tile
    assert plan(0, 1, 1, type_, scale, b_rows, 16, 16, 1) == -1 and plan(1, 1, 17, type_, scale, b_rows, 16, 32, 1) == -1
