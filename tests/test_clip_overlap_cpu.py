"""What moe_clip_grads refuses before any device work: outputs that share memory
with one another or with a gradient that is read - in rows, not only in first
elements - and a norm inside the list.  Slices that interleave are not refused."""

import ctypes
import itertools
import random

import pytest
import torch

from src import _lib


class Desc(ctypes.Structure):
    _fields_ = [("inp", ctypes.c_void_p), ("out", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("in_ld", ctypes.c_int64), ("out_ld", ctypes.c_int64), ("in_type", ctypes.c_int32),
                ("out_type", ctypes.c_int32)]


FAR = 1 << 30


def clip(*tensors, nbytes=8, given=None, norm=FAR, ws=FAR + 4096):
    """Tensors (in, out, rows, cols, in_ld, out_ld, in_type, out_type); with a workspace too small, -4 where the list is taken."""
    d = (Desc * len(tensors))(*[Desc(*t) for t in tensors])
    return _lib.lib().moe_clip_grads(d, len(tensors), 2, 1.0, given, norm, ws, nbytes, None)


def f32(out, rows, cols, ld, inp=None):
    """In place unless `inp` is given."""
    return (out if inp is None else inp, out, rows, cols, ld, ld, 0, 0)


def test_column_slices():
    m = 4096                                                       # a matrix of 50 rows of 64 f32
    col = lambda a, b: f32(m + 4 * a, 50, b - a, 64)  # noqa: E731
    assert clip(col(0, 20), col(10, 30)) == clip(col(10, 30), col(0, 20)) == -1
    assert b"share memory" in _lib.lib().moe_last_error()
    assert clip(col(0, 20), col(20, 64)) == clip(col(40, 64), col(0, 20), col(20, 40)) == -4
    assert clip(col(0, 20), col(19, 64)) == clip(col(0, 64), col(63, 64)) == -1
    row = lambda r: f32(m + 256 * r, 1, 64, 64)  # noqa: E731
    assert clip(col(0, 20), row(3)) == clip(row(49), col(63, 64)) == -1     # a whole row of it, dense
    assert clip(col(0, 20), row(50)) == -4
    assert clip(col(0, 20), f32(m + 256 * 3 + 80, 1, 44, 44)) == -4        # the rest of one of its rows
    # Slices that run into the next row (of another view of the matrix).
    assert clip(col(0, 20), f32(m + 4 * 60, 49, 5, 64)) == -1 and clip(col(0, 20), f32(m + 4 * 60, 49, 4, 64)) == -4
    # Every other row, as rows twice as far apart.
    assert clip(f32(m, 25, 64, 128), f32(m + 256, 25, 64, 128)) == clip(f32(m, 25, 64, 128), f32(m + 256, 49, 8, 128)) == -4
    assert clip(f32(m, 25, 64, 128), col(63, 64)) == -1


def test_outputs_against_gradients():
    a, b = 4096, 8192
    assert clip(f32(b, 1, 10, 10, a), f32(a, 1, 10, 10, b)) == -1          # each the other's output
    assert b"gradient" in _lib.lib().moe_last_error()
    assert clip(f32(b, 1, 10, 10, a), f32(b, 1, 10, 10)) == -1
    assert clip(f32(a + 4, 1, 10, 10, a)) == clip(f32(a, 1, 10, 10, a + 4)) == -1      # shifted against itself
    assert clip(f32(a + 40, 1, 10, 10, a)) == clip(f32(a, 1, 10, 10)) == -4
    assert clip(f32(a, 8, 4, 16, a + 16)) == -4                            # from one slice of a matrix to the next
    assert clip((a, a + 40, 1, 20, 20, 20, 0, 1)) == -1                    # bytes, not elements, count
    assert clip((a, a + 80, 1, 20, 20, 20, 1, 0), (a, b, 1, 20, 20, 20, 1, 0)) == -4   # one gradient to two outputs: 40 bytes
    assert clip(f32(a + 40, 1, 10, 10, a), f32(a + 36, 0, 10, 10)) == -4   # no elements, no memory


def test_a_norm_inside_the_list():
    a, b = 4096, 8192
    take = {"nbytes": 1 << 20}
    assert clip(f32(a, 1, 10, 10), norm=a + 36, **take) == clip(f32(b, 1, 10, 10, a), norm=a, **take) == -1
    assert clip(f32(b, 1, 10, 10, a), norm=b + 8, **take) == clip(f32(b, 1, 10, 10, a), given=b + 8, **take) == -1
    assert b"norm" in _lib.lib().moe_last_error()
    assert clip(f32(a, 1, 10, 10), given=a) == clip(f32(a, 4, 2, 8), given=a + 36) == -1


def test_lists_at_random():
    """Against the elements' addresses one by one."""
    rng = random.Random(1)
    hit = 0
    for _ in range(4000):
        base, n = 4096, rng.randint(1, 4)
        tensors, writes, reads = [], [], []
        for i in range(n):
            rows, cols = rng.randint(1, 4), rng.randint(1, 5)
            ld = cols + rng.choice((0, 1, 3, 7))
            it, ot = rng.choice((0, 1)), rng.choice((0, 1))
            at = base + 4 * rng.randint(0, 30 * n)
            if rng.random() < 0.5:
                t, ot, old = (at, at), it, ld
            else:
                t, old = (base + 4 * rng.randint(0, 30 * n), at), cols + rng.choice((0, 2, 5))
                if t[0] == t[1]:
                    continue
            tensors.append((*t, rows, cols, ld, old, it, ot))
            size = (4, 2)
            writes.append({at + (r * old + c) * size[ot] + x for r in range(rows) for c in range(cols) for x in range(size[ot])})
            reads.append(set() if t[0] == t[1] else
                         {t[0] + (r * ld + c) * size[it] + x for r in range(rows) for c in range(cols) for x in range(size[it])})
        if not tensors:
            continue
        bad = any(writes[i] & writes[j] for i, j in itertools.combinations(range(len(writes)), 2))
        bad = bad or any(writes[i] & reads[j] for i in range(len(writes)) for j in range(len(writes)))
        hit += bad
        assert clip(*tensors) == (-1 if bad else -4), tensors
    assert 400 < hit < 3600


def test_long_lists_out_of_order():
    """Dense neighbours in random order, and interleaved slices of one matrix, stay cheap and accepted."""
    rng = random.Random(2)
    order = list(range(3000))
    rng.shuffle(order)
    assert clip(*[f32(4096 + 40 * i, 1, 10, 10) for i in order]) == -4
    assert clip(*[f32(4096 + 40 * i, 1, 10, 10) for i in order], f32(4096 + 40 * 77 + 36, 1, 1, 1)) == -1
    assert clip(*[f32(4096 + 8 * i, 1000, 2, 1000) for i in order[:] if i < 500]) == -4
    assert clip(*[f32(1 << 24 | 40 * i, 1, 10, 10, 4096 + 40 * i) for i in order]) == -4


def test_python_message_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        from src import grads
        grads.clip_grad_norm([torch.zeros(4)], 1.0, out=[torch.zeros(4)])
