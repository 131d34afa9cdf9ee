"""The stream kernels' work queues (csrc/slx_kernels.hip: TicketQueue) at their edges, through the C ABI on the GPU: queues with fewer items
than waves, launches of changing geometry queued back to back with no synchronisation between them (each must find its counters at
zero), and planes too close together for the kernels' DMA addressing, which stay with the strip kernel."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch


def small_spec(synth, name, w, h):
    spec = dict(synth.make_spec(name))
    spec["width"], spec["height"] = w, h
    spec["calib"] = synth.scaled_calibration(w, h, spec["proj_width"])
    return spec


@pytest.mark.parametrize("name,kernel", [("C2", "slx_stream_kernel<"), ("REF", "slx_gstream_kernel:")])
def test_launches_back_to_back_find_their_counters_at_zero(api, oracle, synth, torch_cuda, name, kernel):
    """One row group up to some dozens, items of 2 to 16 rows, 24 launches in a row on one stream, one synchronisation at the end."""
    torch = torch_cuda
    spec = small_spec(synth, name, 320, 35)
    H, W = spec["height"], spec["width"]
    planes = [synth.random_planes(spec, seed=600 + s) for s in range(6)]
    refs = [oracle.pipeline(spec, p, g, want=("z",))["z"] for p, g in planes]
    ph = torch.from_numpy(np.stack([p for p, _ in planes])).cuda()
    gr = torch.from_numpy(np.stack([g for _, g in planes])).cuda() if name == "REF" else None
    side = torch.cuda.Stream()
    launches = [(n, rows) for n in (1, 6, 2, 5) for rows in (2, 16, 3)] * 2
    z = [torch.full((n, H, W), -7.0, dtype=torch.float64, device="cuda") for n, _ in launches]
    torch.cuda.synchronize()
    with api.Context(spec) as ctx:
        ctx.decode_batch(2, ph[:2], None if gr is None else gr[:2], z[3][:2])    # a batch: the context gets its queue counters
        ctx.synchronize()
        for (n, rows), out in zip(launches, z):
            ctx.set_tuning(stream=2, stream_rows=rows)
            ctx.decode_batch(n, ph[:n], None if gr is None else gr[:n], out, stream=side.cuda_stream)
            assert ctx.last_kernel().startswith(kernel), ctx.last_kernel()
        torch.cuda.synchronize()
        for (n, rows), out in zip(launches, z):
            for k in range(n):
                assert np.array_equal(out[k].cpu().numpy(), refs[k], equal_nan=True), (n, rows, k)


@pytest.mark.parametrize("name", ["C2", "REF"])
def test_planes_closer_than_256_bytes_stay_with_the_strip_kernel(api, oracle, synth, torch_cuda, name):
    """The stream kernels step from plane to plane by the DMA's immediate offset, which needs 256 bytes between planes; a 16 x 8 image has
    128.  Asked for whenever possible, the stream kernel is not possible there, and the depth is the oracle's."""
    torch = torch_cuda
    spec = small_spec(synth, name, 16, 8)
    n = 300
    planes = [synth.random_planes(spec, seed=900 + s) for s in range(n)]
    ph = torch.from_numpy(np.stack([p for p, _ in planes])).cuda()
    gr = torch.from_numpy(np.stack([g for _, g in planes])).cuda() if name == "REF" else None
    z = torch.full((n, 8, 16), -7.0, dtype=torch.float64, device="cuda")
    torch.cuda.synchronize()
    with api.Context(spec) as ctx:
        ctx.set_variant(2)
        ctx.set_tuning(stream=2)
        ctx.decode_batch(n, ph, gr, z)
        ctx.synchronize()
        assert ctx.last_kernel().startswith("slx_strip_kernel<"), ctx.last_kernel()
    for k in range(n):
        assert np.array_equal(z[k].cpu().numpy(), oracle.pipeline(spec, *planes[k], want=("z",))["z"], equal_nan=True), k
