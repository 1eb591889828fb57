"""Workspaces that a caller hands in: used where they hold the bytes in one piece."""

import pytest
import torch

from test_gpu_tree_decode import Case


def test_what_serves_as_scratch():
    from multiscreen import ops
    whole = torch.zeros(64, dtype=torch.float32)
    assert ops._scratch(whole, 256, "cpu") is whole and ops._scratch(whole[8:], 100, "cpu").data_ptr() == whole[8:].data_ptr()
    # one element seen many times, every second one, too few bytes, none
    for x in (whole[:1].expand(1 << 20), whole[::2], whole, None):
        got = ops._scratch(x, 1000, "cpu")
        assert got is not x and got.numel() == 1000 and got.is_contiguous()


@pytest.mark.gpu
def test_scratch_of_tree_and_decode_steps():
    from multiscreen import ops
    case = Case(2, 8, 2, 64, torch.bfloat16, torch.bfloat16, [3000, 2500], "tree", w=(100.0, 4000.0), seed=12)
    d = [x.to("cuda") for x in (case.q, case.kc, case.vc, case.r, case.w)]
    n, par = torch.tensor(case.lengths, device="cuda"), case.parents.to("cuda")
    room = torch.zeros(1 << 23, dtype=torch.uint8, device="cuda")
    views = (None, room, room[:64], room[:1].expand(1 << 23), room[::2])

    def tree(ws):
        return ops.tree_decode(d[0], d[1], d[2], n, par, d[3], d[4], workspace=ws)

    def step(ws):
        return ops.decode_step(d[0][:, 0], d[1], d[2], 2500, d[3], d[4], workspace=ws)

    for call in (tree, step):
        base = call(None)
        assert all(torch.equal(call(x), base) for x in views)
