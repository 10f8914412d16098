"""Tensors with gaps that lie on each other's elements, as clip_gradients takes them: found
from addresses, sizes and strides alone, so without a GPU."""
import random

import pytest
import torch

from ozaki_triton_amd import _lib
from ozaki_triton_amd.gradients import _through_copies


def _elements(t):
    """The bytes of every element."""
    at = [t.data_ptr()]
    for size, stride in zip(t.shape, t.stride()):
        at = [a + i * stride * t.element_size() for a in at for i in range(size)]
    return [frozenset(range(a, a + t.element_size())) for a in at]


def _shared(ins, outs):
    """The same from the bytes themselves."""
    for i, o in enumerate(outs):
        mine = _elements(o)
        every = [b for e in mine for b in e]
        if len(every) != len(set(every)):
            return True
        others = [t for j, pair in enumerate(zip(ins, outs)) if j != i for t in pair]
        if any(set(every) & e for t in others for e in _elements(t)):
            return True
    return False


def _in_place(*tensors):
    return list(tensors), list(tensors)


BASE = torch.zeros(64, 48)
FLAT = torch.zeros(4000)


@pytest.mark.parametrize("ins, outs", [
    _in_place(BASE, BASE[:, ::2]),                          # a part of the other
    _in_place(BASE[:, :4], BASE[:, 2:6]),                   # columns that overlap
    _in_place(BASE[:8], BASE[::2]),                         # some rows of it
    _in_place(BASE[::2], BASE[:8].mT),
    _in_place(BASE[:, ::2], BASE[:, ::2]),                  # the same twice
    _in_place(FLAT[::4], FLAT[1::6], FLAT[2::6]),           # 4 i = 6 j + 2
    _in_place(FLAT.as_strided((5, 5), (3, 2))),             # an element twice
    _in_place(FLAT[:1].expand(5)),
    ([torch.zeros(64, 4), torch.zeros(64, 4)], [BASE[:, :4], BASE[:, 2:6]]),
    ([torch.zeros(64, 4), BASE[:, 3:9]], [BASE[:, :4], torch.zeros(64, 6)]),
    ([torch.zeros(64, 4), BASE], [BASE[:, :4], torch.zeros(64, 48)]),
    # halves of 32-bit elements
    ([torch.zeros(64, 4), torch.zeros(64, 4, dtype=torch.bfloat16)],
     [BASE[:, :4], BASE.view(torch.bfloat16)[:, 7:11]]),
])
def test_shared_elements_are_refused(ins, outs):
    assert _shared(ins, outs)
    with pytest.raises(AssertionError, match="share memory"):
        _through_copies(ins, outs)


@pytest.mark.parametrize("tensors", [
    (BASE[:30, :20], BASE[:30, 20:47], BASE[40:].mT, BASE[31:39, ::2], BASE[31:39, 1::2]),
    (BASE[::2], BASE[1::2]),
    (FLAT[::4], FLAT[1::6], FLAT[3::12]),
    (FLAT[:0], FLAT[:0], FLAT[5:5 + 4 * 9:4].view(3, 3), FLAT[6:40:4]),
    tuple(torch.zeros(100, 200, 3)[:, i, :] for i in range(200)),
    (FLAT.as_strided((7, 5, 3), (200, 13, 4)), FLAT.as_strided((7, 5, 3), (200, 13, 4), 1)),
    (BASE.view(torch.bfloat16)[:, ::2], BASE.view(torch.bfloat16)[:, 1::2]),
])
def test_elements_apart_are_taken(tensors):
    assert _through_copies(*_in_place(*tensors))[2]


def test_inputs_may_share():
    """Only results must be apart; a tensor's own result may lie on it as it likes."""
    square = torch.zeros(20, 20)
    _through_copies([square[:, ::2], square[:, ::2]], [torch.zeros(20, 10), torch.zeros(20, 10)])
    _through_copies([FLAT[:1].expand(7, 5)], [torch.zeros(5, 7).mT])
    _through_copies([square], [square.mT])


def test_against_the_bytes():
    """Views of a few hundred elements, drawn: exactly the lists that share are refused."""
    m = _lib.torch_binding()
    rng = random.Random(5)
    flat = torch.zeros(400)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        tensors = []
        for _ in range(rng.randint(1, 3)):
            of = flat.view(torch.bfloat16) if rng.random() < 0.3 else flat
            size = [rng.randint(1, 5) for _ in range(rng.randint(1, 3))]
            stride = [rng.choice((1, 2, 3, 4, 6, 8, 10, 12, 20, 24)) for _ in size]
            tensors.append(of.as_strided(size, stride, rng.randint(0, 90)))
        outs = [torch.zeros_like(t) if rng.random() < 0.3 else t for t in tensors]
        want = _shared(tensors, outs)
        assert m.share_memory(tensors, outs) == want, [(t.data_ptr(), t.shape, t.stride()) for t in tensors]
        seen[want] += 1
    assert min(seen.values()) > 300, seen
