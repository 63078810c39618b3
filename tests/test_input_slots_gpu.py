"""A grouping that was announced (dctr_prefetch_ids) and is dropped may still be reading its slot when the slot is rewritten: the new ids must not meet
the old ones' counts.  The announcement is made behind a queue of steps that have not run yet, and the slot is rewritten at once."""
import numpy as np
import pytest
import torch

from oracle import deepctr_oracle as O
from tests.util import dev_batch, make_pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["rewrite", "fill", "cancel", "staging_copy", "predict"])
@pytest.mark.parametrize("B", [256, 4096])
def test_a_slot_rewritten_under_a_dropped_grouping(how, B, dev):
    """Against the same steps without the announcement, by the mean over each variable.  The optimizer is Adagrad with lr = 1e-2: after 20 steps a step is about
    lr / sqrt(20) = 2e-3, so one with wrong rows moves the rows' mean by 1e-4 and more.  The order of the float atomics moves an activation by 1e-7 of its
    scale, which turns the ReLU decision of about 1e-6 of the 4096 x 96 x 21 = 8e6 units computed; each turned one adds or takes one of some 2000 examples
    of random sign, 1 / sqrt(2000) of a step, in one column of 64: 2e-3 / 45 / 64 = 7e-7 of the mean, 6e-6 for all of them; 2e-5 leaves three times that."""
    F, V = 39, 60_000
    b = [O.synth_batch(B, F, V, seed=300 + i) for i in range(3)]
    b[2] = ((b[2][0] + V // 2) % V,) + b[2][1:]                 # other ids than those announced
    pinned = [torch.from_numpy(np.ascontiguousarray(x)).pin_memory() for x in b[2]]
    runs = []
    for hint in (False, True):
        _, _, eng = make_pair("deepfm", B=B, F=F, V=V, K=16, layers=(64, 32), opt="Adagrad", lr=1e-2, seed=3, use_graph=False)
        slots = [tuple(x[:B] for x in eng.input_slot(k)) for k in range(2)]
        for to, of in zip(slots, b):
            for x, y in zip(to, dev_batch(*of, dev)):
                x.copy_(y)
        foreign = dev_batch(*b[2], dev)
        prob = torch.empty(B, device=dev)
        on = 0 if how in ("staging_copy", "predict") else 1      # (foreign buffers are staged into slot 0)
        torch.cuda.synchronize()
        for _ in range(20):
            eng.train_step(*slots[1 - on], want_loss=False)
        if hint:
            eng.prefetch_ids(slots[on][0])
        if how == "fill":
            eng.input_slot_fill(on, *(x.data_ptr() for x in pinned), B)
            eng.input_slot_acquire(on)
            eng.train_step(*slots[on], want_loss=False)
        elif how == "staging_copy":
            eng.train_step(*foreign, want_loss=False)
        elif how == "predict":
            eng.predict(foreign[0], foreign[1], prob, None)
            eng.train_step(*foreign, want_loss=False)
        else:
            if how == "rewrite":
                eng.input_slot_rewrite(on)
            else:
                eng.prefetch_cancel()
            other = torch.cuda.Stream()
            with torch.cuda.stream(other):
                for x, y in zip(slots[on], foreign):
                    x.copy_(y)
            other.synchronize()
            eng.train_step(*slots[on], want_loss=False)
        eng.check_ids()
        runs.append(dict(eng.get_params()))
        eng.close()
    for k, v in runs[0].items():
        assert np.abs(v - runs[1][k]).mean() <= 2e-5, k
