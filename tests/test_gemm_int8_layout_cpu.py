"""Scratch memory for 8-bit operands whose rows are no whole dwords: what the size queries say, without a GPU."""
from aitemplate_amd import _kernels, eager


def test_layout_bytes():
    lib = _kernels.load()
    row = lambda K: (K + 15) // 16 * 16  # noqa: E731
    for M, N, K in [(1, 1, 513), (70, 96, 1024), (777, 2731, 1101), (1 << 20, 5, 131071)]:
        assert lib.aitamd_gemm_int8_layout_bytes(M, N, K) == 4096 + (M + N) * row(K)
        assert lib.aitamd_gemm_int8_layout_bytes(0, N, K) == 4096 + N * row(K)
        assert lib.aitamd_gemm_int8_layout_bytes(M, 0, K) == 4096 + M * row(K)
        assert eager.gemm_int8_workspace_bytes(M, N, K, any_byte=True) >= 4096 + (M + N) * row(K)
    # rows so short that they are multiplied as they lie, and what is refused anyway
    for M, N, K in [(70, 96, 512), (70, 96, 0), (0, 0, 1024), (-1, 5, 1024), (5, 5, 131072)]:
        assert lib.aitamd_gemm_int8_layout_bytes(M, N, K) == 0
    # rows of an odd K are always laid out: both queries say the same
    for K in (514, 1101):
        assert eager.gemm_int8_workspace_bytes(64, 96, K) == eager.gemm_int8_workspace_bytes(64, 96, K, any_byte=True) > 0
    assert eager.gemm_int8_workspace_bytes(2000, 2000, 1024) < eager.gemm_int8_workspace_bytes(2000, 2000, 1024, any_byte=True)
