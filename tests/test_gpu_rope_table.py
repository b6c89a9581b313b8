"""The rotation's table into a caller's plane: into that plane and nothing beside it. GPU only (-m gpu)."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_plane_that_is_given(rq_ctx):
    import torch

    plane = torch.full((12, 64), 3.0, device="cuda")
    assert rq_ctx.rope_table(10, 64, out=plane[1:11]).data_ptr() == plane[1].data_ptr()
    assert torch.equal(plane[1:11], rq_ctx.rope_table(10, 64)) and (plane[[0, 11]] == 3.0).all()


def test_planes_that_are_refused(rq_ctx):
    import torch

    plane = torch.zeros((12, 64), device="cuda")
    for out in (plane, plane[:10, :32], plane.double()[:10], torch.zeros((10, 64)), torch.zeros((64, 10), device="cuda").t(), plane[:10].reshape(-1), plane[:9]):
        with pytest.raises(ValueError, match="rope_table"):
            rq_ctx.rope_table(10, 64, out=out)
    rq_ctx.check()
