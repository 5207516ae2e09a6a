"""Captures that others have in progress while runtimes come and go: they record on, and what they
recorded replays."""
import os
import subprocess
import sys
import threading

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

MODES = [(m, s) for m in ("thread_local", "global") for s in (True, False)]


def beside(mode, same_thread, what):
    """A stream is captured, and `what` is called meanwhile by this thread or another one; whatever comes of
    it, torch's current stream is the one from before."""
    import torch

    stream, graph, x = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode=mode)
        try:
            x += 1
            if same_thread:
                what()
            else:
                t = threading.Thread(target=what)
                t.start()
                t.join()
            x += 1
        finally:
            graph.capture_end()  # (raises where something has ended the capture)
    torch.cuda.synchronize()
    for n in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert x.tolist() == [2.0 * n] * 4


def used(rt):
    """A runtime that holds workspaces, cached blocks and loaded kernels, and two buffers of its own."""
    import numpy as np
    import rxla_amd as rx

    q, kv = rt.zeros((2, 8, 128), rx.DType.F32), rt.zeros((2, 2, 3000, 128), rx.DType.BF16)
    y = rx.grouped_query_attention(rt, q, kv, kv, rt.buffer(np.array([3000, 5], np.int32)))
    rt.synchronize()
    return [q, y]


@pytest.mark.parametrize("mode,same_thread", MODES)
def test_a_runtime_is_created(rt, mode, same_thread):
    import rxla_amd as rx

    made = []
    beside(mode, same_thread, lambda: made.append(rx.Runtime(0)))
    assert used(made[0])


FIRST = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
from test_gpu_captures import beside, used
import torch
torch.zeros(1, device="cuda")
import rxla_amd as rx
made = []
beside({mode!r}, {same!r}, lambda: made.append(rx.Runtime(0)))
assert used(made[0])
print("right")
"""


@pytest.mark.parametrize("mode,same_thread", MODES)
def test_the_first_runtime_of_a_process_is_created(mode, same_thread):
    """(which sets up what all runtimes of a device share)"""
    code = FIRST.format(root=ROOT, tests=os.path.join(ROOT, "tests"), mode=mode, same=same_thread)
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert got.returncode == 0 and "right" in got.stdout, got.stderr[-2000:]


@pytest.mark.parametrize("mode,same_thread", MODES)
@pytest.mark.parametrize("last", ["runtime", "buffer"])
def test_a_runtime_is_released(rt, mode, same_thread, last):
    """By its owner, or with the last of its buffers: as the collector may, at any time."""
    import rxla_amd as rx

    own = rx.Runtime(0)
    bufs = used(own)
    if last == "buffer":
        own.close()

    def release():
        for b in bufs:
            b.release()
        own.close()

    beside(mode, same_thread, release)


def decoder(rt):
    import numpy as np
    from decoder_fixtures import tiny_params
    from test_gpu_decoder import build, small_cfg

    cfg = small_cfg()
    model = build(rt, cfg, tiny_params(cfg), 2)
    model.generate(rt.buffer(np.zeros((2, 3), np.int32)), 5)  # (a graph of its step)
    rt.synchronize()
    return model


def hybrid(rt):
    import numpy as np
    from oracle import qwen35
    from test_gpu_qwen35 import CONFIGS, build

    cfg = CONFIGS["tiny"]
    model = build(rt, cfg, qwen35.random_params(cfg, seed=1, std=0.05))
    for _ in range(3):
        model.forward(rt.buffer(np.zeros((1, 4), np.int32)))
    rt.synchronize()
    return model


@pytest.mark.parametrize("mode,same_thread", MODES)
@pytest.mark.parametrize("make", [decoder, hybrid])
def test_a_model_is_released(rt, mode, same_thread, make):
    beside(mode, same_thread, make(rt).close)
