"""The largest batches and vocabularies of msa_verify: what a launch cannot hold is refused with a
reason.  On the CPU, where a call that is taken fails at its launch."""

import pytest
import torch


def test_launches_fit_their_grids():
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would start a kernel")
    from multiscreen import _native
    L = _native.lib()

    def verify(B, M, V, greedy):
        need = L.msa_verify_workspace_bytes(B, M, V, greedy)
        return L.msa_verify(_native.pack_verify_args(16, M * V, V, 0, 0, 0, 16, 0, 0, 0 if greedy else 16, 16, 16, 16,
                                                     16 if greedy else 0, need, B, M, V, 0), None)

    # a block of 1024 threads a sequence, of 256 a row and part of 8192 entries: fewer than 2^32 threads along x,
    # 65535 blocks along y
    for args, taken in (((2 ** 22 - 1, 1, 10, 0), True), ((2 ** 22, 1, 10, 0), False), ((2 ** 24, 1, 10, 0), False),
                        ((2 ** 20, 64, 10, 0), True), ((2 ** 18, 63, 10, 1), True), ((2 ** 18, 64, 10, 1), False),
                        ((2 ** 24, 1, 10, 1), False), ((2 ** 24 - 1, 1, 10, 1), True), ((1, 1, 65535 * 8192, 1), True),
                        ((1, 1, 65535 * 8192 + 1, 1), False), ((1, 1, 2 ** 31 - 1, 0), True)):
        rc = verify(*args)
        assert rc == (3 if taken else 1), (args, rc)
        assert taken or "at most" in L.msa_last_error().decode()
