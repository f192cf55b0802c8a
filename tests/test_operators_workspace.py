"""The workspaces' documented bounds (include/naju_loss.h, include/naju_mixer.h),
over the whole range of rows."""
import random

from naju_amd import _lib


def _up(n, m):
    return -(-n // m) * m


def _log(rng, lo, hi):
    return int(lo * (hi / lo) ** rng.random())


def _parts(d, rows):
    return (10 if d >= 256 else 64) * 4 * d * rows + 4096


def _head(n, d, v):
    """The documented bound, rounded up by a page for the regions' alignment."""
    dl = min(2 * n * _up(v, 256), max(1 << 30, 512 * n))
    columns = min(v, max(256, (1 << 30) // (2 * n) // 256 * 256))
    pieces = -(-v // columns)
    return dl + 2 * n * _up(d, 8) + 4 * n + (4 * n * d if pieces > 1 else 0) + _parts(d, max(n, columns))


def _gated(n, d, f):
    return 4 * n * _up(f, 32) + _parts(d, max(n, 2 * _up(f, 32)))


def test_head():
    size = _lib.lib().naju_linear_xent_workspace_bytes
    # most rows served: 16 GiB of them the piece of 256 columns
    assert 512 << 25 <= size(1 << 25, 64, 50257, 1) <= _head(1 << 25, 64, 50257)
    assert size(1 << 21, 64, 50257, 1) <= (1 << 30) + 6 * 64 * (1 << 21) + (1 << 24)
    rng = random.Random(3)
    for _ in range(20000):
        n, d, v = _log(rng, 1, 1 << 25), _log(rng, 1, 1 << 14), _log(rng, 1, 1 << 18)
        assert size(n, d, v, 1) <= _head(n, d, v), (n, d, v)


def test_gated():
    size = _lib.lib().naju_gated_workspace_bytes
    rng = random.Random(4)
    for _ in range(20000):
        n, d, f = _log(rng, 1, 1 << 24), _log(rng, 1, 1 << 14), _log(rng, 1, 1 << 16)
        assert 4 * n * f <= size(n, d, f) <= _gated(n, d, f), (n, d, f)
    # few rows: the parts are most of it
    assert 4 * 64 * 5504 * 6 < size(64, 2048, 5504)
