"""GPU: what the kernels report through the device status word, from the first call of a process on."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HEAD = """
import threading
import time
import torch
from dlcompiler_b200 import _lib, check_device_status, shared_prefix_attention_fwd, sink_attention_fwd
dev = torch.device("cuda:0")
k = torch.randn(4, 16, 1, 64, device=dev).bfloat16()
q, o = k[0, :1].clone(), torch.empty(1, 1, 64, dtype=k.dtype, device=dev)
table, lens, start, one = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([[0, 1]], [30], [0], [1]))
own = torch.tensor([[2]], dtype=torch.int32, device=dev)

def sinks():
    sink_attention_fwd(q, k, k, o, table, start, one, lens, 1, 100, 0)

def prefix():
    shared_prefix_attention_fwd(q, k, k, o, table, lens, torch.stack([start, one]).flatten(), own, one)

def reported():
    try:
        check_device_status()
    except _lib.DlblasError as e:
        assert "row 0, column 1 of a block table names page 9" in str(e), e
        return True
    return False

torch.cuda.synchronize()
"""


def _fresh(code):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", HEAD + code + "print('through')"], cwd=root, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0 and "through" in res.stdout, res.stdout + res.stderr


@pytest.mark.parametrize("call", ["sinks", "prefix"])
def test_first_call_under_capture(cuda_device, call):
    """Nothing is reported before a replay, a replay's bad page is, and a replay takes back no other call's."""
    _fresh(f"""
call = {call}
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call()
assert not reported()
graph.replay()
assert not reported()
table[0, 1] = 9
graph.replay()
assert reported() and not reported()
call()
table[0, 1] = 1
graph.replay()
assert reported() and not reported()
""")


def test_first_call_from_two_threads(cuda_device):
    """Both get the same word, however long it takes to make one."""
    _fresh("""
slow = torch.zeros
torch.zeros = lambda *a, **kw: (slow(*a, **kw), time.sleep(0.5))[0]
gate, words = threading.Barrier(2), []

def first():
    gate.wait()
    words.append(_lib.status_word(dev))

threads = [threading.Thread(target=first) for _ in range(2)]
[t.start() for t in threads], [t.join() for t in threads]
assert len(words) == 2 and words[0].data_ptr() == words[1].data_ptr() == _lib.status_word(dev).data_ptr()
assert words[0].tolist() == [0] * 4
""")


def test_check_waits_for_other_streams(cuda_device):
    """A bad page behind a tenth of a second of other work on a stream that is not the current one."""
    _fresh("""
table[0, 1] = 9
sinks()
assert reported()
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    torch.cuda._sleep(200_000_000)
    sinks()
assert reported()
table[0, 1] = 1
""")
