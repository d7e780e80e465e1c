"""Which scratch attention takes (kernels/_launch.py), without a GPU: one per
stream, and one of its own for each capture."""
import torch

from qlinear.kernels import _launch


def test_a_capture_never_gets_the_streams_scratch(monkeypatch):
    cpu, size = torch.device("cpu"), 2 * _launch._SCRATCH_HEADER
    now = [0]
    monkeypatch.setattr(_launch, "is_capturing", lambda: now[0] != 0)
    monkeypatch.setattr(_launch, "current_device", lambda: None)         # the index of torch.device("cpu")

    class Lib:
        ql_capture_id = staticmethod(lambda stream: now[0])
    monkeypatch.setattr(_launch._lib, "load", lambda: Lib)
    eager = _launch.scratch(cpu, 77, size)
    assert _launch.scratch(cpu, 77, size) is eager and int(eager.count_nonzero()) == 0
    held = [eager]
    for capture in (5, 6):
        now[0] = capture
        buf = _launch.scratch(cpu, 77, size)
        assert all(buf is not h for h in held) and int(buf[:_launch._SCRATCH_HEADER].count_nonzero()) == 0
        assert _launch.scratch(cpu, 77, size) is buf                     # one a capture
        assert _launch.scratch(cpu, 78, size) is not buf                 # and stream
        held.append(buf)
    now[0] = 0
    assert _launch.scratch(cpu, 77, size) is eager
    for stream in (77, 78):
        _launch._scratches.pop((None, stream), None)
        _launch._graph_scratches.pop((None, stream), None)
