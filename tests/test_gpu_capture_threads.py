"""The learner's graphs are recorded while other threads of the process use the GPU's events, as RCCL's watchdog does."""
import threading

import numpy as np
import pytest
import torch

import rl_gan_amd as R

pytestmark = pytest.mark.gpu


def _learner():
    L = R.CuriousLearner(R.LearnerConfig(n_env=64, batch_size=64, memory_capacity=256, seed=3))
    L.fill()
    return L


def test_another_thread_queries_an_event_during_the_capture():
    L, plain = _learner(), _learner()
    done = torch.cuda.Event()
    done.record()
    torch.cuda.synchronize()
    seen, tail = [], L._tail_body

    def query():
        try:
            seen.append(done.query())
        except Exception as e:                                  # (kept for the assertion: it would be lost with the thread)
            seen.append(e)

    def tail_with_a_query(*a):
        if torch.cuda.is_current_stream_capturing():
            t = threading.Thread(target=query)
            t.start()
            t.join()
        return tail(*a)

    L._tail_body = tail_with_a_query
    L.capture()                                                 # (two eager iterations first)
    for _ in range(4):
        L.step()
    for _ in range(6):
        plain.step()
    assert seen == [True, True]
    assert L.losses() == plain.losses() and np.array_equal(L.actor.e.get_flat(), plain.actor.e.get_flat())
