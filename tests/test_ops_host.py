"""The host side of msplat.ops, without a GPU."""
import contextlib

import pytest

torch = pytest.importorskip("torch")


class FakeStream:
    device, cuda_stream = torch.device("cuda", 1), 0x1230


def test_status_asks_on_the_streams_device(monkeypatch):
    """The failure counters belong to a device: status makes its stream's current."""
    from msplat import ops
    entered, asked = [], []

    @contextlib.contextmanager
    def device(d):
        entered.append(torch.device("cuda", d) if isinstance(d, int) else d)
        yield
        entered.pop()

    class Lib:
        @staticmethod
        def msplat_ops_status(handle):
            asked.append((handle, list(entered)))
            return 0
    monkeypatch.setattr(ops, "_lib", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "device", device)
    ops.status(FakeStream())
    assert asked == [(0x1230, [torch.device("cuda", 1)])] and not entered


def test_rehearsals_are_refused_by_number():
    from msplat import ops
    L = ops._lib()
    for kernels in (-1, 3):
        assert L.msplat_ops_rehearse_timeout(kernels, None) == 1
        assert "kernels must be" in L.msplat_last_error().decode()
