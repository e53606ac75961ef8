"""The attentions over a paged cache where a slip shows: every key counted once, and running maxima that move.

Counting: key i is 32 e[i % 128] and its value e[(i // 128) % 128]; a query 32 e[j] gives the keys i = j (mod 128) the score
90.5 and the others 0, weights of 1 and of under 2^-126. So the output tells how many of these keys were counted for every
(i // 128) % 128, c of B: c / B, rounded once (2^-8) behind weights and sums in fp32 (2^-12). c is 3 at most, so a key that
is lost, or counted twice, moves it by a quarter or more. All j are asked.

Moving maxima: scores rise by 6.5, more than a running maximum lets pass before it moves (8 ln 2 = 5.5), at one key of every
second tile of 128, beside 128 and more keys at the height before: what was gathered before the move keeps a weight of a
few tenths. Rows in turn follow the rise, half of it, its reverse, or nothing. Tolerance: the output's rounding, 2^-8 |o|;
the weights', 2^-8 A with A = sum p |v|, and 2^-12 A for their exponential and sums; twice A times the error of a score s in
fp32, 128 * 2^-24 sum |q_i k_i| / sqrt(128) for the products and 2^-22 |s| for its difference from the maximum.
"""

import math

import pytest
import torch

from ipe_b200 import _native as nat
from test_gpu_paged import DEV, HALF, Batch, decode, normal, prefill, shared

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------- every key

def counted(batch):
    """The cache's keys and values as their positions name them."""
    eye = torch.eye(128, dtype=torch.bfloat16, device=DEV)
    for s, n in enumerate(batch.length):
        pages, rows = batch.places(s)
        i = torch.arange(n, device=DEV)
        batch.k[pages, :, rows] = 32 * eye[i % 128][:, None]
        batch.v[pages, :, rows] = eye[i // 128 % 128][:, None]
    return batch


def check_counts(attention, batch, q_heads):
    group = q_heads // batch.kv_heads
    sees = torch.cat([torch.arange(n - m + 1, n + 1) if n else torch.zeros(m, dtype=torch.int64)
                      for m, n in zip(batch.new, batch.length)]).to(DEV)[:, None, None]
    row, head = torch.arange(len(sees), device=DEV)[:, None], torch.arange(q_heads, device=DEV)[None]
    value, eye = torch.arange(128, device=DEV), 32 * torch.eye(128, dtype=torch.bfloat16, device=DEV)
    for ask in range(0, 128, group):
        j = (ask + head % group + 5 * row) % 128
        out = attention(batch, eye[j]).view(len(sees), q_heads, 128).double()
        of = (sees - j[..., None] + 127).div(128, rounding_mode="floor").clamp(min=0)
        count = of // 128 + (value < of % 128).long()
        count = torch.where(of == 0, (value == 0).long(), count)  # none of these keys: all weigh alike, in values e[0]
        o = torch.where(sees > 0, count / of.clamp(min=1).double(), 0.0)
        assert bool(((out - o).abs() <= (HALF + 2.0 ** -12) * o + 2.0 ** -100).all()), ask
    assert nat.device_error() == 0


@pytest.mark.parametrize(("lengths", "page", "q_heads", "kv_heads"), [
    ([1], 16, 16, 8),
    ([640], 16, 16, 8),
    ([63, 64, 65, 127, 128, 129, 0, 1], 16, 4, 1),
    ([5000, 1, 0, 300], 64, 40, 8),
    ([9000, 1, 100, 4000], 128, 28, 4),
    (list(range(300, 360)), 32, 32, 8),
    ([33000, 5, 12000], 16, 7, 1),
    ([20000] + [150] * 30, 32, 16, 8),
])
def test_decode_counts_every_key(lengths, page, q_heads, kv_heads):
    check_counts(decode, counted(Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=1)), q_heads)


@pytest.mark.parametrize(("new", "past", "page", "q_heads", "kv_heads"), [
    ([127, 129, 1, 64], [0, 0, 0, 0], 32, 16, 8),
    ([300, 17, 1], [0, 1000, 4000], 64, 8, 2),
    ([65, 1, 200], [63, 128, 700], 128, 28, 4),
    ([513], [2000], 16, 8, 1),
    ([40], [30000], 32, 16, 8),
    ([70, 3, 130], [9000, 12000, 0], 16, 6, 2),
    ([(37 * n) % 211 for n in range(40)], [(91 * n) % 517 for n in range(40)], 16, 24, 8),  # whole blocks, many per CTA
])
def test_prefill_counts_every_key(new, past, page, q_heads, kv_heads):
    check_counts(prefill, counted(Batch(new, past, page, kv_heads, seed=2)), q_heads)


@pytest.mark.parametrize(("lengths", "prefix", "page", "q_heads", "kv_heads"), [
    ([33, 40, 64], 2, 16, 16, 8),
    ([700 + 3 * n for n in range(20)], 40, 16, 16, 8),
    ([1300 + n % 50 for n in range(130)], 20, 64, 40, 8),
    ([513 + 128 * n for n in range(9)], 4, 128, 3, 1),
    ([8200, 8193, 6000, 12000], 64, 128, 12, 2),
])
def test_shared_prefix_counts_every_key(lengths, prefix, page, q_heads, kv_heads):
    b = counted(Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=3, prefix=prefix))
    check_counts(shared, b, q_heads)


# ---------------------------------------------------------------------------------- moving maxima

RISE, FOLLOWS = 6.5, (1.0, 0.0, -1.0, 0.5, 1.0, 0.9)


def rising(batch, seed, most=8):
    """Keys whose part along a direction of their KV head rises with the position, values with a mean of their tile."""
    direction = normal((batch.kv_heads, 128), seed).sign().float()
    for s, n in enumerate(batch.length):
        pages, rows = batch.places(s)
        i = torch.arange(n, device=DEV)
        tile = i // 128
        height = RISE * (tile // 2 + ((tile % 2 == 1) & (i % 128 == 37 * tile % 128)).long()).clamp(max=most)
        shape = (n, batch.kv_heads, 128)
        along = height[:, None, None] * (math.sqrt(128) / 128) * direction
        batch.k[pages, :, rows] = (0.3 * normal(shape, seed + 1).float() + along).bfloat16()
        mean = normal((n // 128 + 1, batch.kv_heads, 128), seed + 2)[tile].float()
        batch.v[pages, :, rows] = (0.3 * normal(shape, seed + 3).float() + mean).bfloat16()
    return batch, direction


def follow(batch, direction, q_heads, seed):
    """Queries that follow the rise, each row and head in its own way."""
    group = q_heads // batch.kv_heads
    which = torch.arange(batch.tokens, device=DEV)[:, None] + torch.arange(q_heads, device=DEV) // 2
    along = torch.tensor(FOLLOWS, device=DEV)[which % len(FOLLOWS)][..., None] * direction.repeat_interleave(group, 0)
    return (0.3 * normal((batch.tokens, q_heads, 128), seed).float() + along).bfloat16()


def check_moves(out, batch, q, keys=None):
    """Against the definition in 64 bits; the share of rows whose maximum moves behind their first tile (of `keys` keys)."""
    heads, at, rows, moved = q.shape[1], 0, 0, 0
    got = out.view(len(out), heads, 128).double()
    for s, n in enumerate(batch.new):
        total = batch.length[s]
        for h in range(heads):
            k, v = batch.keys(s, h // (heads // batch.kv_heads), total)
            x = q[at:at + n, h].double()
            score = x @ k.T / math.sqrt(128)
            hidden = torch.arange(total, device=DEV) > (total - n + torch.arange(n, device=DEV))[:, None]
            score = score.masked_fill(hidden, -math.inf)
            p = torch.softmax(score, -1)
            o, a = p @ v, p @ v.abs()
            error = 128 * 2.0 ** -24 * (x.abs() @ k.abs().T / math.sqrt(128)).amax(-1) + 2.0 ** -22 * score.nan_to_num(0, 0, 0).abs().amax(-1)
            limit = HALF * o.abs() + (HALF + 2.0 ** -12 + 2 * error[:, None]) * a
            assert float(((got[at:at + n, h] - o).abs() - limit).max()) <= 0, (s, h)
            if n and h < 8:
                use = total if keys is None else min(keys, total)
                tops = torch.nn.functional.pad(score[:, :use], (0, -use % 128), value=-math.inf).view(n, -1, 128).amax(-1)
                top, any_ = tops[:, 0], torch.zeros(n, dtype=torch.bool, device=DEV)
                for t in range(1, tops.shape[1]):
                    move = tops[:, t] > top + 8 * math.log(2)
                    top, any_ = torch.where(move, tops[:, t], top), any_ | move
                rows, moved = rows + n, moved + int(any_.sum())
        at += n
    assert nat.device_error() == 0
    return moved / rows


@pytest.mark.parametrize(("new", "past", "page", "q_heads", "kv_heads"), [
    ([900], [0], 16, 4, 2),
    ([300, 700], [0, 40], 64, 3, 1),
    ([260, 100], [700, 333], 128, 10, 2),
    ([70, 9, 1], [3000, 900, 700], 32, 16, 8),  # in runs: parts with other maxima
    ([20], [9000], 16, 7, 1),
    ([150] * 20, [500] * 20, 32, 16, 8),  # whole blocks
])
def test_prefill_of_rising_scores(new, past, page, q_heads, kv_heads):
    b, direction = rising(Batch(new, past, page, kv_heads, seed=4), 10)
    q = follow(b, direction, q_heads, 20)
    assert 0.1 < check_moves(prefill(b, q), b, q) < 0.9


@pytest.mark.parametrize(("lengths", "prefix", "page", "q_heads", "kv_heads"), [
    ([700 + 3 * n for n in range(20)], 40, 16, 16, 8),
    ([1300 + n % 50 for n in range(40)], 20, 64, 40, 8),
    ([900 + 128 * n for n in range(9)], 6, 128, 3, 1),
    ([3000 + n for n in range(150)], 23, 128, 4, 2),
])
def test_shared_prefix_of_rising_scores(lengths, prefix, page, q_heads, kv_heads):
    b, direction = rising(Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=5, prefix=prefix), 30)
    q = follow(b, direction, q_heads, 40)
    assert 0.1 < check_moves(shared(b, q), b, q, keys=prefix * page) < 0.9


@pytest.mark.parametrize(("lengths", "page", "q_heads", "kv_heads"), [([900, 700, 130, 300], 16, 16, 8), ([6000, 800], 64, 5, 1)])
def test_decode_of_rising_scores(lengths, page, q_heads, kv_heads):
    b, direction = rising(Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=6), 50)
    q = follow(b, direction, q_heads, 60)
    check_moves(decode(b, q), b, q)


@pytest.mark.parametrize(("new", "past", "page", "q_heads", "kv_heads"), [([900], [0], 16, 4, 2), ([70, 9, 1], [3000, 900, 700], 32, 16, 8)])
def test_prefill_of_rising_scores_and_large_values(new, past, page, q_heads, kv_heads):
    """Values of about 2^116: weights of up to 256 beside a maximum that has not moved take the accumulators past fp32's
    range, weights of at most 1 do not."""
    b, direction = rising(Batch(new, past, page, kv_heads, seed=7), 70, most=3)
    b.v *= 2.0 ** 116
    q = follow(b, direction, q_heads, 80)
    out = prefill(b, q)
    assert torch.isfinite(out).all()
    check_moves(out, b, q)
