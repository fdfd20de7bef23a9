"""The device status word reaches ``read_status`` whoever makes a call first and however: eagerly, inside a capture,
under ``torch.compile``."""

import subprocess
import sys

import pytest
import torch

import recipes
from conftest import ROOT
from triton_mla import _lib, mla_decode, read_status
from triton_mla.kernel import _status_word

pytestmark = pytest.mark.gpu


def _run(code):
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT / "triton-mla_b200", capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_the_word_is_the_librarys(device):
    import ctypes

    word = ctypes.c_void_p()
    assert _lib.load().tmla_status_word(ctypes.byref(word)) == 0
    t = _status_word(device)
    assert t.data_ptr() == word.value and t.dtype == torch.int32 and t.device == device
    read_status(device)
    t.fill_(_lib.STATUS_TIMEOUT)
    assert read_status(device, reset=False) == _lib.STATUS_TIMEOUT
    assert read_status(device) == _lib.STATUS_TIMEOUT and read_status(device) == 0


def test_first_linear_int8_inside_a_capture_reports_its_status():
    """A process whose first call is captured: the call gets the word, which outlives the graph and its pool."""
    _run("""
import torch
from triton_mla import layer_ops, read_status
from triton_mla.kernel import _status_word
device = torch.device("cuda", 0)
q = torch.ones(40, 64, device=device, dtype=torch.int8)
s = torch.ones(40, device=device)
op, seen = torch.ops.triton_mla.linear_int8, []
def spy(*args):
    seen.append(args[-1])
    return op(*args)
torch.ops.triton_mla.linear_int8 = spy
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = layer_ops.linear_int8(q, s, q, s, torch.float32)
assert seen[0] is not None and seen[0].data_ptr() == _status_word(device).data_ptr()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, torch.full_like(y, 64.0)) and read_status() == 0
_status_word(device).fill_(2)          # as a timed-out wait of the replayed call would
graph.replay()
assert read_status(reset=False) == 2, "a replay does not clear it"
del graph, y
torch.cuda.empty_cache()
assert read_status() == 2 and read_status() == 0
""")


def test_first_decode_inside_a_capture_keeps_its_status():
    """The same for the decode: no replay clears the word (it would, if the word were made within the capture)."""
    _run("""
import torch
from triton_mla import mla_decode, read_status
from triton_mla.kernel import _status_word
device = torch.device("cuda", 0)
q = torch.randn(2, 16, 576, device=device, dtype=torch.bfloat16)
kv = torch.randn(4, 64, 576, device=device, dtype=torch.bfloat16)
lens = torch.tensor([100, 64], device=device, dtype=torch.int32)
bt = torch.tensor([[0, 1], [2, 3]], device=device, dtype=torch.int32)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = mla_decode(q, kv, lens, bt, num_splits=1)
graph.replay()
assert read_status() == 0
bt[0, 0] = 10_000_000
graph.replay()
bt[0, 0] = 0
graph.replay()
assert read_status() == 1
""")


def test_a_compiled_decode_reports_a_bad_page(device):
    case = recipes.paged_case([200, 50], 16, 64, seed=41)
    q, kv, lens, bt = (case[k].to(device) for k in ("q", "kv", "seqlens", "block_table"))

    @torch.compile(fullgraph=True, backend="aot_eager")
    def f(q, kv, lens, bt):
        return mla_decode(q, kv, lens, bt, num_splits=1)

    read_status(device)
    want = mla_decode(q, kv, lens, bt, num_splits=1)
    assert torch.equal(f(q, kv, lens, bt), want) and read_status(device) == 0
    bt = bt.clone()
    bt[0, 1] = 10_000_000
    got = f(q, kv, lens, bt)
    assert read_status(device) == _lib.STATUS_BAD_PAGE and torch.equal(got[1], want[1])
