"""Clipping refuses a factor that lies in what it writes. (On a machine with a GPU only the refusals are made: the addresses are no memory.)"""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from multigputrainmlp_b200 import _lib  # noqa: E402
from test_layer_norm_refusals import entries  # noqa: E402

A, B = (0x1000, 10, 0), (0x2000, 30, 1)  # 40 bytes and 60
FAR = [(0x9000, 10, 0), (0xa000, 30, 1)]


def clip(result, rows=(A, B), out=None):
    place = lambda r: ctypes.cast(entries(*r), ctypes.c_void_p)  # noqa: E731
    return int(_lib.load().mgt_launch_clip_gradients(place(rows), len(rows), result, place(out) if out else None, None))


def test_the_factor_lies_beside_what_is_written():
    for inside in (0xffc, 0x1000, 0x1004, 0x1020, 0x1024, 0x1ffc, 0x2000, 0x2030, 0x2038):
        assert clip(inside) == 1 and clip(inside, (B, A)) == 1 and clip(inside, FAR, [A, B]) == 1, hex(inside)
    if not torch.cuda.is_available():  # what fits reaches the launch, which has no device here
        for beside in (0xff8, 0x1028, 0x1ff8, 0x203c, 0x4000):
            assert clip(beside) == 4 and clip(beside, (B, A)) == 4 and clip(beside, FAR, [A, B]) == 4, hex(beside)
        assert clip(0x1000, (A, B), FAR) == 4  # (it may lie in what is only read)
        assert clip(0x1000, ((0x1000, 0, 0), B)) == 4 and clip(0x1000, ((None, 0, 0),)) == 4
