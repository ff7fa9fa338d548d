"""Which gradients share memory: the clipping's own answer against the sets of their elements, for layouts with gaps too."""
import random

import pytest
import torch

from transformer_amd import grad_clip


def shared(grads):
    try:
        grad_clip._refuse_shared("clip_grad_norm_", grads)
    except ValueError:
        return True
    return False


def elements(t):
    """The bytes of ``t``, one number each."""
    at = torch.zeros((), dtype=torch.int64)
    for s, n in zip(t.stride(), t.shape):
        at = at.unsqueeze(-1) + s * torch.arange(n)
    es = t.element_size()
    return ((at.reshape(-1, 1) * es + torch.arange(es)).reshape(-1) + t.data_ptr()).tolist()


BUF = torch.zeros(40, 24)
CASES = {
    "the same with gaps twice": ([BUF[:, 3:17], BUF[:, 3:17]], True),
    "windows that overlap": ([BUF[:, :4], BUF[:, 2:6]], True),
    "windows side by side": ([BUF[:, :4], BUF[:, 4:9], BUF[:, 9:]], False),
    "windows of other rows": ([BUF[:20, 3:17], BUF[20:, 3:17]], False),
    "rows that one window shares": ([BUF[:21, 3:17], BUF[20:, 5:8]], True),
    "a run within the gaps": ([BUF[:, :8], BUF.view(-1)[32:48]], False),
    "a run that reaches a window": ([BUF[:, :8], BUF.view(-1)[32:49]], True),
    "every second element, and the others": ([BUF[:, ::2], BUF[:, 1::2]], False),
    "every second and every third": ([BUF[:, ::2], BUF[:, 3::3]], True),
    "other strides": ([BUF[:, :4], BUF.view(80, 12)[:, 4:8]], False),
    "other strides that meet": ([BUF[:, :4], BUF.view(80, 12)[:, 3:8]], True),
    "a transpose": ([BUF[:, :4], BUF.t()[4:]], False),
    "a transpose that meets": ([BUF[:, :4].t(), BUF[:, 3:]], True),
    "no elements": ([BUF[:, :0], BUF[:, :4], BUF[:0, :4]], False),
    "rows that overlap themselves": ([BUF.view(-1).as_strided((5, 4), (2, 1))], True),
    "two types in one buffer": ([BUF[:, :4], BUF.view(torch.bfloat16)[:, 8:]], False),
    "two types that meet": ([BUF[:, :4], BUF.view(torch.bfloat16)[:, 7:]], True),
}


@pytest.mark.parametrize("name", sorted(CASES))
def test_known_layouts(name):
    grads, want = CASES[name]
    assert shared(grads) == shared(grads[::-1]) == want


def test_layouts_at_random():
    rng, seen = random.Random(7), [0, 0]
    for _ in range(1500):
        grads = []
        for _ in range(rng.choice([2, 2, 2, 3])):
            buf = BUF.view(torch.bfloat16) if rng.random() < 0.3 else BUF
            t = buf.reshape(rng.choice([(40, -1), (20, -1), (8, 10, -1), (-1,), (4, 5, 4, -1)]))
            for d in range(t.dim()):
                a, b = sorted(rng.randrange(t.size(d) + 1) for _ in range(2))
                if rng.random() < 0.7:
                    t = t.narrow(d, a, b - a)
                if rng.random() < 0.2:
                    t = t[(slice(None),) * d + (slice(None, None, rng.choice([2, 3])),)]
            grads.append(t.permute(rng.sample(range(t.dim()), t.dim())))
        every = [e for t in grads for e in set(elements(t))]
        want = len(every) != len(set(every))
        seen[want] += 1
        assert shared(grads) == want, [(t.data_ptr() - BUF.data_ptr(), t.shape, t.stride(), t.dtype) for t in grads]
    assert min(seen) > 200


def test_many_rows_of_one_buffer_are_compared_at_once():
    buf = torch.zeros(1 << 20, 4)
    steps, meet = [], grad_clip._meet

    def counted(*a):
        steps.append(1)
        return meet(*a)

    grad_clip._meet = counted
    try:
        assert not shared([buf[:, :1], buf[:, 1:3], buf[:, 3:]])
    finally:
        grad_clip._meet = meet
    assert len(steps) < 20
