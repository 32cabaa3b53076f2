"""Which windows the engine says overflowed their token buffers: the decoder leaves a batch's counts, then its flags,
one entry per window of the batch, whatever the engine's capacity."""
from __future__ import annotations

import numpy as np
import pytest


class _Done:
    def synchronize(self):
        pass


@pytest.mark.parametrize("batch", [1, 3, 4])
def test_flags_of_a_batch(pk, batch):
    import torch

    capacity = 4
    eng = pk.engine.ParakeetEngine.__new__(pk.engine.ParakeetEngine)
    eng.capacity, eng.max_tokens = capacity, 6
    meta = torch.full((2 * capacity,), 1, dtype=torch.int32)  # what an earlier, larger batch left
    counts, flags = np.arange(batch) + 3, np.arange(batch) % 2
    meta[:batch], meta[batch:2 * batch] = torch.from_numpy(counts), torch.from_numpy(flags)
    eng._slots = [dict(tokens=torch.zeros((3, capacity, 6), dtype=torch.int32), meta=meta, done=_Done())]
    got = eng._collect((0, batch))
    assert [len(tok) for tok, *_ in got] == np.minimum(counts, 6).tolist()
    assert [over for *_, over in got] == (flags == 1).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("alternatives", [None, 2])
def test_windows_that_overflow_say_so(pk, device, alternatives):
    """Token buffers that hold the shorter windows alone: in batches of every size, a full one before smaller ones."""
    package = pk.synthetic.make_package("fp16", seed=0)
    package.update(pk.synthetic.make_decoder("fp16", seed=0))
    pcm = pk.synthetic.make_pcm(60.0, seed=9)
    plans = pk.windows.plan_stateless_windows(len(pcm))
    windows = [(pcm[p.source_start_sample:p.source_end_sample], p) for p in plans][:4]
    assert len(windows) == 4
    eng = pk.engine.ParakeetEngine(device, package, "fp16", capacity=4)
    try:
        lengths = [len(r.tokens) for r in eng.transcribe_windows(windows)]
    finally:
        eng.destroy()
    most = sorted(set(lengths))[len(set(lengths)) // 2] - 1  # some windows fit, some do not
    assert min(lengths) <= most < max(lengths)
    eng = pk.engine.ParakeetEngine(device, package, "fp16", capacity=4, max_tokens=most, alternatives=alternatives)
    try:
        for first, last in ((0, 4), (0, 1), (1, 4), (2, 4), (0, 3), (3, 4)):
            got = eng.transcribe_windows(windows[first:last])
            assert [r.overflow for r in got] == [n > most for n in lengths[first:last]]
            assert [len(r.tokens) for r in got] == [min(n, most) for n in lengths[first:last]]
    finally:
        eng.destroy()
