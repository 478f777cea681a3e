"""Host-side logic of the batch operators (no GPU)."""

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from asdsl_b200 import _lib
    from asdsl_b200.build import build_library

    build_library()
    return _lib


def test_plan_step_refuses_inputs_that_it_would_overwrite(lib):
    """CTAs read the inputs while another writes the outputs, so the two must be apart (checked before any launch)."""
    # three requests, four free pages, a table [3][2], four tokens; addresses far apart
    at = dict(kv=0x1000, new=0x2000, free=0x3000, table=0x4000, cu=0x5000, total=0x6000, slots=0x7000, pos=0x8000, req=0x9000,
              counts=0xA000)

    def step(**kw):
        a = {**at, **kw}
        lib.call("asdsl_b200_plan_step", a["kv"], a["new"], 3, a["free"], 4, 16, a["table"], 2, 2, a["cu"], a["total"], a["slots"],
                 a["pos"], a["req"], 4, a["counts"], None)

    for kw in (dict(kv=at["total"]), dict(kv=at["total"] + 8), dict(new=at["total"]), dict(new=at["cu"] + 12), dict(free=at["slots"]),
               dict(kv=at["table"] + 20), dict(kv=at["pos"] - 8), dict(new=at["req"] + 12), dict(free=at["counts"] + 8)):
        with pytest.raises(ValueError, match="overlap"):
            step(**kw)


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
