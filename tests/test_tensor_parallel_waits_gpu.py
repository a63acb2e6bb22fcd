"""Tensor-parallel ranks that share a process or a GPU: who waits for whom, and what a wait in vain becomes."""
import ctypes as C
import threading
import time

import numpy as np
import pytest

import golden_cases as GC
from ctranslate2_amd import _lib
from test_tensor_parallel_gpu import _model_dir, _sources

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(120)]


@pytest.mark.parametrize("late", (0, 1))
@pytest.mark.parametrize("beam", (1, 4))
def test_a_late_rank_in_the_same_process(gpu, beam, late):
    """One rank has done all it can alone for a second before the other's session starts, with its allocations
    and blocking copies: no kernel of the first may be waiting for it (streams of one process share hardware
    queues), and the results are the unsharded engine's."""
    import ctranslate2_amd as ct2
    path, cfg, src = _model_dir("tiny"), GC.SYNTHETIC["tiny"], _sources("tiny")
    kw = dict(beam_size=beam, max_decoding_length=cfg["max_len"], min_decoding_length=cfg["min_len"],
              return_scores=True)
    single = ct2.Translator(path, compute_type="int8")
    want, scores = single.translate_ids(src, **kw)
    ranks = ct2.Translator.tensor_parallel_local(path, 2, compute_type="int8")
    for r, t in enumerate(ranks):
        assert t.tensor_parallel_info() == {"rank": r, "world": 2, "mailboxes": False, "backend": "in-process"}
    got, errors = [None, None], []

    def work(r):
        try:
            time.sleep(1.0 if r == late else 0.0)
            got[r] = ranks[r].translate_ids(src, **kw)
        except Exception as e:  # noqa: BLE001 - raised below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=90)
    assert not errors, errors
    for hyps, s in got:
        assert hyps == want and np.array_equal(s, scores)
    for t in ranks:
        t.close()


def test_one_shot_exchanges_beside_many_streams(gpu):
    """The self test finds two streams whose kernels run together whatever other streams the process holds."""
    import torch
    streams = [torch.cuda.Stream() for _ in range(9)]
    for s in streams:
        with torch.cuda.stream(s):
            torch.zeros(4, device="cuda").add_(1)
    torch.cuda.synchronize()
    us = C.c_float()
    _lib.check(_lib.lib().ct2x_tp_selftest_oneshot(0, 2, C.c_int64(32), C.c_int64(256), C.c_int64(512), 20,
                                                   C.byref(us)))
    assert us.value > 0
