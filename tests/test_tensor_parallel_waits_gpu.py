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


RANK = """
import json, sys
import numpy as np
import ctranslate2_amd as ct2
model, rank, segment, sources, steps = sys.argv[1], int(sys.argv[2]), sys.argv[3], json.loads(sys.argv[4]), 4
t = ct2.Translator.tensor_parallel_shm(model, rank, 2, segment, compute_type="int8")
kw = dict(beam_size=2, max_decoding_length=8, min_decoding_length=8)
tgt = np.ones((len(sources), steps), np.int32)
same = [s[:1] for s in sources]
t.translate_ids(sources, **kw)
t.step_logits(same, tgt)
t.debug_give_up_exchanges()
errors = []
for call in (lambda: t.translate_ids(sources, **kw), lambda: t.translate_ids(sources, beam_size=1, **{
        k: v for k, v in kw.items() if k != "beam_size"}), lambda: t.step_logits(same, tgt)):
    try:
        call()
        errors.append("")
    except ct2.Ct2xError as e:
        errors.append(str(e))
print("ERRORS " + json.dumps(errors))
t.close()
"""


def test_a_wait_in_vain_is_an_error(gpu):
    """A poll that gave up (marked by the host on both ranks, so that no kernel waits) makes every call that hands
    out results fail: greedy and beam search, logits."""
    import json
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    segment = "ct2x_tp_give_up_%d" % os.getpid()
    env = dict(os.environ, HSA_ENABLE_IPC_MODE_LEGACY="0", PYTHONPATH=root)
    procs = [subprocess.Popen([sys.executable, "-c", RANK, _model_dir("tiny"), str(r), segment,
                               json.dumps(_sources("tiny"))], env=env, cwd=root, stdout=subprocess.PIPE,
                              stderr=subprocess.PIPE, text=True) for r in range(2)]
    try:
        outs = [p.communicate(timeout=60) for p in procs]
    finally:
        for p in procs:
            p.kill()
    for p, (out, err) in zip(procs, outs):
        assert p.returncode == 0, err[-2000:]
        errors = json.loads(next(line for line in out.splitlines() if line.startswith("ERRORS "))[7:])
        assert len(errors) == 3 and all("did not arrive" in e for e in errors), errors


def test_give_up_needs_mailboxes(gpu):
    import ctranslate2_amd as ct2
    path = _model_dir("tiny")
    for t in [ct2.Translator(path)] + ct2.Translator.tensor_parallel_local(path, 2):
        with pytest.raises(ct2.Ct2xError, match="tensor-parallel rank|no mailboxes"):
            t.debug_give_up_exchanges()
        t.close()


def test_streams_asked_of_a_rank_are_one(gpu):
    """num_streams splits a batch into sessions that run at once; a rank's exchanges meet the others' in the order of
    one session, so a tensor-parallel rank takes the sub-batches together."""
    import ctranslate2_amd as ct2
    path, cfg, src = _model_dir("tiny"), GC.SYNTHETIC["tiny"], _sources("tiny")
    kw = dict(beam_size=2, max_decoding_length=cfg["max_len"], min_decoding_length=cfg["min_len"],
              return_scores=True, num_streams=3)
    single = ct2.Translator(path, compute_type="int8")
    want, scores = single.translate_ids(src, **kw)
    ranks = ct2.Translator.tensor_parallel_local(path, 2, compute_type="int8")
    got = [None, None]

    def work(r):
        got[r] = ranks[r].translate_ids(src, **kw)

    threads = [threading.Thread(target=work, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=90)
    for hyps, s in got:
        assert hyps == want and np.array_equal(s, scores)
    for t in ranks:
        t.close()
