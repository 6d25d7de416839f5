"""How many shares of dx the device chooses (vloss_rows_grad_kernel), restated: never more than the launch has blocks for, where a block
computes one share (the CUDA-core forms), and never more rows of shares than there is room for."""
import random

import pytest

MOST = 32


def _up(a, b):
    return (a + b - 1) // b


def few_work(tokens, vocab, width):
    piece = min(max((64 << 20) // (4 * tokens) // 128 * 128, 1024), _up(vocab, 4) * 4)
    tiles = _up(tokens, 128) * _up(width, 128)
    room = max(1, min(MOST, _up(8 * 148, tiles)))
    return dict(workers=148, rows=8 if tokens <= 8 else 16, acc=1, ht=_up(width, 512), vt=0, steps=_up(piece, 64), step=64, room=room, tokens=tokens, most=room, dw=False)


def any_work(tokens, vocab, width):
    w = few_work(tokens, vocab, width)
    piece = min(max((64 << 20) // (4 * tokens) // 128 * 128, 1024), _up(vocab, 4) * 4)
    return dict(w, workers=2 * 148, rows=128, ht=_up(width, 128), steps=_up(piece, 16), step=16)


def tc_work(tokens, vocab, width):
    rows = _up(tokens, 256) * 256
    n = max((256 << 20) // (2 * rows) // 256 * 256, 8192)
    piece = _up(_up(vocab, _up(vocab, n)), 256) * 256
    room = max(1, min(MOST, _up(8 * 74, rows // 256 * _up(width, 256))))
    return dict(workers=74, rows=256, acc=256, ht=_up(width, 256), vt=_up(piece, 256), steps=piece // 64, step=64, room=room, tokens=rows, most=MOST, dw=True)


def chosen(work, n, capped=True):
    best = None
    for s in range(1, MOST + 1):
        mt, W = _up(n, work["rows"]), work["workers"]
        dx, dw = mt * work["ht"] * s, work["vt"] * work["ht"] if work["dw"] else 0
        dx_cost, dw_cost = _up(work["steps"], s) + 12, _up(n, work["step"]) + 4
        more = dx % W
        fewer = W - more
        x = min(dx_cost // dw_cost, dw // fewer) if more else 0
        rest = dw - x * fewer
        last = rest % W
        busy = (dx // W + 1) * dx_cost + (rest // W + (last > fewer)) * dw_cost if more else 0
        idle = dx // W * dx_cost + (x + rest // W + (last > 0)) * dw_cost
        fits = s == 1 or ((not capped or s <= work["most"]) and s * (_up(n, work["acc"]) * work["acc"]) <= work["room"] * work["tokens"]
                          and work["steps"] >= 8 * s)
        if fits and (best is None or max(busy, idle) < best[0]):
            best = max(busy, idle), s
    return best[1]


def _sizes(form, rng):
    few = form is few_work
    return (rng.randint(1, 32) if few else int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 18)),
            8 * int(2 ** rng.uniform(0, 11)) if few else int(2 ** rng.uniform(0, 14)))


@pytest.mark.parametrize("form", [few_work, any_work, tc_work])
def test_every_share_is_computed_and_has_room(form):
    rng, over = random.Random(4), 0
    for _ in range(4000):
        tokens, vocab, width = _sizes(form, rng)
        work, n = form(tokens, vocab, width), rng.randint(0, tokens)
        s = chosen(work, n)
        assert s <= work["most"] and s * (_up(n, work["acc"]) * work["acc"]) <= work["room"] * work["tokens"]
        over += chosen(work, n, capped=False) > work["most"]
    assert (over > 0) == (form is not tc_work)              # the limit is needed, and reached, where a block computes one share
