"""Calls of several host threads on one stream share its workspace, and most
entries pass data through it from one kernel to the next: each call's launches
have to be queued without another's between them."""
from __future__ import annotations

import ast
import threading
import time
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

BINDINGS = Path(__file__).resolve().parents[1] / "cublade_amd" / "bindings" / "hip"


def _attribute_calls(node, name):
    return [n for n in ast.walk(node) if isinstance(n, ast.Call)
            and isinstance(n.func, ast.Attribute) and n.func.attr == name]


def test_every_workspace_is_taken_under_its_lock():
    """In every binding, workspace() and the library call that gets it stand in
    one `with` block that holds workspace_lock()."""
    found = 0
    for path in sorted(BINDINGS.glob("*.py")):
        tree = ast.parse(path.read_text())
        held = []
        for node in ast.walk(tree):
            if isinstance(node, ast.With) and any(_attribute_calls(i.context_expr, "workspace_lock")
                                                  for i in node.items):
                held += [n for s in node.body for n in ast.walk(s)]
        for call in _attribute_calls(tree, "workspace"):
            assert call in held, f"{path.name}:{call.lineno}"
            found += 1
        for use in [n for n in ast.walk(tree) if isinstance(n, ast.Name) and n.id == "ws"
                    and isinstance(n.ctx, ast.Load)]:
            assert use in held, f"{path.name}:{use.lineno}"
    assert found >= 9


@pytest.mark.parametrize("streams", [1, 2])
def test_calls_on_one_stream_take_turns(monkeypatch, streams):
    """attend_kv from two threads against a library whose call takes a while:
    never two at once on one stream; on two streams they do not wait."""
    from cublade_amd import _abi
    from cublade_amd.bindings.hip import kv_cache as kvb
    dev = torch.device("cpu")
    inside, most, gate = [], [], threading.Barrier(2)
    mine = threading.local()

    def attend(*args):
        inside.append(mine.stream)
        most.append(inside.count(mine.stream))
        if streams == 2 and not mine.met:      # both threads are here, or this times out
            mine.met = True
            gate.wait(timeout=20)
        time.sleep(0.02)
        inside.remove(mine.stream)
        return 0

    monkeypatch.setattr(_abi, "_ws", {(0, i): torch.zeros(1 << 16, dtype=torch.uint8) for i in (0, 1)})
    monkeypatch.setattr(_abi, "device_index", lambda d: 0)
    monkeypatch.setattr(_abi, "stream_handle", lambda d: mine.stream)
    monkeypatch.setattr(_abi, "lib", lambda: SimpleNamespace(
        cbq_kv_attend_ws_bytes=lambda *a: 1 << 16, cbq_kv_attend=attend))
    view = _abi.KvCache(4096, 4096, 4096, 4096, 4, 1, 16, 16, _abi.KV_INT8)
    q = torch.zeros(1, 1, 16, dtype=torch.float16)
    one = torch.ones(1, dtype=torch.int32)
    errors = []

    def work(stream):
        try:
            mine.stream, mine.met = stream, False
            for _ in range(3):
                kvb.kv_attend(view, dev, q, one[None], one)
        except Exception as e:       # reported below: a thread's own exceptions are not seen
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i % streams,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert len(most) == 6 and max(most) == 1


@pytest.mark.gpu
def test_two_threads_on_one_stream():
    """attend_kv with split keys from two threads on the default stream, of
    different inputs: every result has the bits of a call alone."""
    from cublade_amd.quantization import attend_kv
    from tests import _kv
    g = torch.Generator(device="cuda").manual_seed(41)
    cases = []
    for lens in ([9000, 40], [7000, 8000]):
        table, pages = _kv.make_table(lens, 64, g)
        cache = _kv.random_cache(pages, 2, 128, 64, torch.int8, g)
        q = torch.randn(2, 8, 128, generator=g, device="cuda").bfloat16()
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cases.append((q, cache, table, n))
    want = [attend_kv(*c) for c in cases]
    torch.cuda.synchronize()
    got, start = [[], []], threading.Barrier(2)

    def work(i):
        start.wait(timeout=60)
        for _ in range(200):
            got[i].append(attend_kv(*cases[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 200
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_the_watched_status_is_read_under_the_lock():
    """With CUBLADE_CHECK_EXCHANGE=1 a call clears its workspace's status word,
    runs, and reads the word: another thread's call in between would clear what
    this one has to report."""
    found = 0
    for path in sorted(BINDINGS.glob("quantize_*.py")):
        tree = ast.parse(path.read_text())
        held = [n for node in ast.walk(tree) if isinstance(node, ast.With)
                and any(_attribute_calls(i.context_expr, "workspace_lock") for i in node.items)
                for s in node.body for n in ast.walk(s)]
        for call in [n for n in ast.walk(tree) if isinstance(n, ast.Call) and isinstance(n.func, ast.Name)
                     and n.func.id in ("watch_exchange", "check_exchange")]:
            assert call in held, f"{path.name}:{call.lineno}"
            found += 1
    assert found == 4
