"""Calls and graphs over a 4-bit pool that run at the same time on different streams."""
import threading

import numpy as np
import pytest
import torch

import serving_engine_b200 as b200
from serving_engine_b200 import q4
from serving_engine_b200.e2e import random_llama
from serving_engine_b200.q4_serve import Q4Batch
from tests.test_q4_gpu import DEV, make_batch, metadata

pytestmark = pytest.mark.gpu


def test_two_batches_decode_on_two_streams():
    """Their graphs hold workspaces of their own: the tokens are those of one after the other."""
    model = random_llama("tiny", 0, torch.bfloat16, DEV)
    rng = np.random.default_rng(0)
    prompts = [[rng.integers(0, 1000, n).tolist() for n in lens] for lens in ((700, 1500, 20), (900, 33, 1200))]
    want = []
    for p in prompts:
        batch = Q4Batch(model, 3, 1600)
        batch.prefill(p)
        want.append(batch.decode(60).tolist())
    for _ in range(3):
        batches = [Q4Batch(model, 3, 1600) for _ in range(2)]
        for batch, p in zip(batches, prompts):
            batch.prefill(p)
            batch.decode(0)  # captures
        held = [q4._workspaces[0, batch._workspace._key] for batch in batches]
        assert held[0][1] != held[1][1] and held[0][0].data_ptr() != held[1][0].data_ptr()
        torch.cuda.synchronize()
        got = [None, None]
        streams = [torch.cuda.Stream() for _ in range(2)]

        def decode(i):
            with torch.cuda.stream(streams[i]):
                got[i] = batches[i].decode(60)

        threads = [threading.Thread(target=decode, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert [g.tolist() for g in got] == want
    b200.check_device_errors()


def test_threads_on_streams_of_their_own():
    """First calls from four threads at once, then many more: each as if alone."""
    batches = [make_batch([3000 + 100 * i, 40, 700], [1, 2, 1], 8, 2, 128, torch.bfloat16, seed=i) for i in range(4)]
    args = [(b["q"], b["pool"][0], b["pool"][1], metadata(b), 8, 2, b["scale"]) for b in batches]
    want = [b200.paged_flash_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    start = threading.Barrier(4)
    bad = []

    def work(i):
        start.wait()
        with torch.cuda.stream(streams[i]):
            outs = [b200.paged_flash_attention(*args[i]) for _ in range(200)]
            streams[i].synchronize()
        bad.extend(i for o, l in outs if not (torch.equal(o, want[i][0]) and torch.equal(l, want[i][1])))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    b200.check_device_errors()
