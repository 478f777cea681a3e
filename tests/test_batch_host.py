"""Host-side logic of the batch operators (no GPU)."""

import pytest
import torch


@pytest.fixture
def workspace(monkeypatch):
    """An AttentionWorkspace on the CPU whose sizes are the calls' tokens in bytes."""
    from asdsl_b200.kernels import paged

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged.AttentionWorkspace, "_size", lambda self, device, entry, *key: 1000 + max(key))
    return paged.AttentionWorkspace()


def test_outgrown_workspace_buffers_stay(workspace):
    """A graph captured on a workspace holds its buffers' addresses: a larger call must not free them."""
    import weakref

    cpu = torch.device("cpu")
    first = [weakref.ref(workspace.sized(cpu, 8, 8, 8, 8)), weakref.ref(workspace.merge(cpu, 8, 8, 8))]
    again = workspace.sized(cpu, 4, 4, 4, 4), workspace.merge(cpu, 8, 8, 8)
    assert again[0] is first[0]() and again[1] is first[1]()  # smaller calls use them
    del again
    assert workspace.sized(cpu, 5000, 5000, 8, 8).numel() >= 6000 and workspace.merge(cpu, 9000, 8, 8).numel() >= 10000
    assert first[0]() is not None and first[1]() is not None


def test_workspace_growth_adds_up(workspace):
    """Calls that grow a little each time do not each leave a buffer behind."""
    cpu = torch.device("cpu")
    for n in range(1, 20000, 7):
        ws = workspace.sized(cpu, n, n, 1, 1)
    held = sum(t.numel() for t in workspace._outgrown)
    assert ws.numel() >= 20990 and held <= 2 * ws.numel()


def test_stream_workspaces_are_bounded(monkeypatch):
    """Streams that come and go do not each keep a workspace for good; a stream in use keeps its own."""
    from asdsl_b200.kernels import paged

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged, "_stream_workspaces", {})
    for stream in range(200):
        monkeypatch.setattr(paged, "_raw_stream", lambda index, s=stream: s)
        ws = paged._workspace(torch.device("cuda", 0))
        assert paged._workspace(torch.device("cuda", 0)) is ws
    assert len(paged._stream_workspaces) <= 32
