"""`stream` has to be a torch stream of the operands' GPU: the launch would go to another
stream than the one given otherwise, and run beside what it waits for."""
import pytest

torch = pytest.importorskip("torch")


class _Elsewhere:
    """Looks like a stream of a second GPU."""
    def __init__(self):
        self.device, self.cuda_stream = torch.device("cuda", 1), 0
        self.stream_id, self.device_index, self.device_type = 0, 1, 1


@pytest.mark.gpu
@pytest.mark.parametrize("wrong", [_Elsewhere, lambda: 0, lambda: "side"])
def test_stream_of_another_gpu(S, wrong):
    h = lambda *s: torch.zeros(s, dtype=torch.half, device="cuda")  # noqa: E731
    x, offsets = h(4, 8), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    r, stream = S.route(x, 2), wrong()
    xs = h(8, 8)
    for call in (lambda: S.route(x, 2, stream=stream),
                 lambda: S.route_backward(x, r, r.weights, stream=stream),
                 lambda: S.group_entries(r.experts, 8, stream=stream),
                 lambda: S.dispatch(x, r, stream=stream), lambda: S.combine(xs, r, stream=stream),
                 lambda: S.dispatch_backward(xs, r, stream=stream),
                 lambda: S.combine_backward(x, xs, r, stream=stream),
                 lambda: S.grouped_mm(x, h(1, 4, 8), offsets, stream=stream),
                 lambda: S.grouped_mm_backward(x, x, h(1, 8, 8), offsets, stream=stream),
                 lambda: S.adapter_mm(x, h(4, 8), h(1, 2, 8), h(1, 4, 2), offsets[:1].repeat(4),
                                      stream=stream)):
        with pytest.raises(S.SpmmError) as e:
            call()
        assert e.value.code == S.SPMM_INVALID and "stream" in str(e.value)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert S.dispatch(x, r, stream=side).shape == (8, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert S.dispatch(x, r, stream=torch.cuda.current_stream()).shape == (8, 8)
