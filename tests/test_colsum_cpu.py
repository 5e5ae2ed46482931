"""How the column sums (bias gradients) are split, and what their C entry refuses (no GPU needed)."""
from vilmedic_amd._lib import lib


def test_rows_are_split_over_enough_workgroups_and_scratch_stays_small():
    L = lib()
    for rows, cols in ((12544, 768), (50176, 64), (8192, 30528), (12544, 1)):
        parts = L.vm_colsum_bf16_ws(rows, cols) // (4 * cols)
        groups = -(-cols // 256)
        assert parts * groups >= min(98, rows // 128) and parts * groups <= max(512, groups) and parts <= 128, (rows, cols, parts)
    assert L.vm_colsum_bf16_ws(1024, 100) == 0 and L.vm_colsum_bf16_ws(1025, 100) == 4 * 9 * 100 and L.vm_colsum_bf16_ws(0, 8) == 0 and L.vm_colsum_bf16_ws(2**31 - 1, 1) == 4 * 128


def test_refusals():
    L = lib()
    fake = 1 << 20                  # a non-null address that is never followed: the refusal is about the numbers
    assert L.vm_colsum_bf16_ex(None, 8, fake, 1, 1, None, None, 0, None) == -1
    assert L.vm_colsum_bf16_ex(fake, 9, fake, 1, 1, None, None, 0, None) == -1
    assert L.vm_colsum_bf16_ex(fake, 768, fake, 12544, 768, None, fake, 100, None) == -1
    assert L.vm_colsum_bf16_ex(fake, 768, fake, 12544, 768, None, fake + 4, 1 << 30, None) == -1
