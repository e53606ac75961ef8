"""What the attentions over a paged cache make of values that are not finite, against the definition.

softmax(s) v with s = q k^T / sqrt(128), in 64 bits: a row that sees a score of +infinity or NaN is NaN throughout. A score of
-infinity has the weight 0, which gives NaN beside a value that is not finite. Elsewhere a weight is above 0, however small,
so an infinite value gives infinity, and NaN beside one of the other sign or a NaN.
"""

import math

import pytest
import torch

from ipe_b200 import _native as nat
from ipe_b200 import ops
from test_gpu_paged import DEV, HALF, NAN, Batch, decode, normal, prefill, shared

pytestmark = pytest.mark.gpu
INF = float("inf")


def attend(batch, q):
    """(o, A) of the definition in 64 bits [tokens, Hq * 128]; A = sum p |v| over the finite values."""
    heads = q.shape[1]
    o = torch.zeros(batch.tokens, heads, 128, dtype=torch.float64, device=DEV)
    a = torch.zeros_like(o)
    at = 0
    for s, n in enumerate(batch.new):
        total = batch.length[s]
        for h in range(heads if total else 0):
            k, v = batch.keys(s, h // (heads // batch.kv_heads), total)
            score = q[at:at + n, h].double() @ k.T / math.sqrt(128)
            hidden = torch.arange(total, device=DEV) > (total - n + torch.arange(n, device=DEV))[:, None]
            score = torch.where(hidden, -INF, score)
            p = torch.softmax(score, -1)
            finite = torch.where(torch.isfinite(v), v, 0.0)
            counted = (score > -INF).double()
            nothing = (~hidden & (score == -INF)).double()
            up, down = counted @ (v == INF).double() > 0, counted @ (v == -INF).double() > 0
            none = (counted @ torch.isnan(v).double() + nothing @ (~torch.isfinite(v)).double() > 0) | (up & down)
            x = torch.where(up, INF, p @ finite)
            x = torch.where(down, -INF, x)
            o[at:at + n, h] = torch.where(none | torch.isnan(p).any(-1, keepdim=True), NAN, x)
            a[at:at + n, h] = p @ finite.abs()
        at += n
    return o.view(batch.tokens, -1), a.view(batch.tokens, -1)


def check(out, batch, q):
    """Equal where the definition is not finite; elsewhere the output's rounding, the weights' and the scores' (as in
    test_gpu_paged.py)."""
    o, a = attend(batch, q)
    got = out[:batch.tokens].double()
    lost = ~torch.isfinite(o)
    assert torch.equal(torch.isnan(got), torch.isnan(o))
    assert torch.equal(got == INF, o == INF) and torch.equal(got == -INF, o == -INF)
    over = ((got - o).abs() - (HALF * o.abs() + (HALF + 2.0 ** -11) * a))[~lost]
    assert over.numel() == 0 or float(over.max()) <= 0
    assert nat.device_error() == 0


def spoil(batch, seed):
    """A few values of every sequence infinite or NaN, in dimensions of their own; the first and the last key's too."""
    g = torch.Generator().manual_seed(seed)
    for s, n in enumerate(batch.length):
        if n == 0:
            continue
        for dim, value in ((0, INF), (1, -INF), (2, NAN), (3, INF), (3, -INF), (4, INF), (4, NAN), (5, INF), (6, -INF)):
            key = {5: 0, 6: n - 1}.get(dim, int(torch.randint(n, (1,), generator=g)))
            pages, rows = batch.places(s, key + 1, key)
            batch.v[pages, :, rows, dim] = value
    return batch


DECODE = [
    ([640], 16, 16, 8),
    ([1, 16, 17, 63, 64, 65, 0, 300], 16, 4, 2),
    ([5000, 1, 700], 64, 40, 8),
    ([20000, 9], 32, 7, 1),
    ([130] * 60, 128, 8, 8),
]


@pytest.mark.parametrize(("lengths", "page", "q_heads", "kv_heads"), DECODE)
def test_decode_of_infinite_values(lengths, page, q_heads, kv_heads):
    b = spoil(Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=7).fill(100), 8)
    q = normal((len(lengths), q_heads, 128), 9, 1.5)
    check(decode(b, q), b, q)


@pytest.mark.parametrize("place", [0, 70, 299])
@pytest.mark.parametrize("step", [1, 6])
def test_decode_of_an_infinite_value_under_any_weight(place, step):
    """Scores from about -150 to 150: an infinite value whose weight is the largest, one whose is below 1e-80, and between."""
    b = Batch([1] * 2, [299, 40], 16, 2, seed=11).fill(200)
    q = normal((2, 4, 128), 12, 4.0)
    pages, rows = b.places(0)
    direction = q[0].view(2, 2, 128).float().mean(1)
    direction /= direction.norm(dim=-1, keepdim=True)
    level = torch.linspace(-40, 40, 300, device=DEV)[torch.arange(300, device=DEV) * step * 49 % 300]
    b.k[pages, :, rows] = (b.k[pages, :, rows].float() * 0.05 + level[:, None, None] * direction).bfloat16()
    b.v[pages[place], :, rows[place], 3] = INF
    b.v[pages[place], 1, rows[place], 4] = -INF
    out = decode(b, q).view(2, 4, 128)
    assert (out[0, :, 3] == INF).all() and (out[0, 2:, 4] == -INF).all()
    bad = ~torch.isfinite(out)
    assert int(bad.sum()) == 6
    assert nat.device_error() == 0


def test_decode_of_scores_that_are_not_finite():
    """Keys with an infinite element: +infinity for some heads, -infinity (and the weight 0) for others."""
    b = Batch([1] * 3, [299, 40, 700], 16, 2, seed=13).fill(300)
    q = normal((3, 6, 128), 14, 1.5)
    for s, key in ((0, 100), (1, 40), (2, 0)):
        pages, rows = b.places(s, key + 1, key)
        b.k[pages, :, rows, 9] = -INF
        if s == 2:
            b.v[pages, 0, rows, 5] = INF
    check(decode(b, q), b, q)


# ----------------------------------------------------------------------- prefill and the shared prefix

PREFILL = [
    ([1, 130], [0, 0], 16, 16, 8),
    ([300, 17, 1, 0], [0, 900, 2000, 30], 64, 8, 2),
    ([257], [0], 128, 5, 1),
    ([100, 100], [129, 31], 16, 6, 2),
    ([90], [5000], 32, 16, 8),
    ([(37 * n) % 211 for n in range(40)], [(91 * n) % 517 for n in range(40)], 16, 24, 8),  # whole blocks, many per CTA
]


@pytest.mark.parametrize(("new", "past", "page", "q_heads", "kv_heads"), PREFILL)
def test_prefill_of_infinite_values(new, past, page, q_heads, kv_heads):
    b = spoil(Batch(new, past, page, kv_heads, seed=15).fill(400), 16)
    q = normal((b.tokens, q_heads, 128), 17, 1.5)
    out = prefill(b, q)
    check(out, b, q)
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(prefill(b, q)))


@pytest.mark.parametrize(("new", "past"), [([200, 70], [30, 500]), ([150] * 40, [20] * 40)])
def test_prefill_of_scores_that_are_not_finite(new, past):
    """A key with an infinite element early in every second sequence, under infinite values too; a NaN query."""
    b = Batch(new, past, 16, 8, seed=18).fill(500)
    q = normal((b.tokens, 16, 128), 19, 1.5)
    for s in range(0, len(new), 2):
        pages, rows = b.places(s, past[s] + 12, past[s] + 11)
        b.k[pages, :, rows, 9] = -INF
        b.v[pages, 0, rows, 5] = INF
    q[new[0] // 2, 3] = NAN
    check(prefill(b, q), b, q)


SHARED = [
    ([33, 40, 64], 2, 16, 16, 8),
    ([32, 31, 1, 0, 33], 2, 16, 4, 2),
    ([700 + 3 * n for n in range(20)], 40, 16, 16, 8),
    ([1300 + n % 50 for n in range(130)], 20, 64, 40, 8),
    ([513 + 128 * n for n in range(9)], 4, 128, 3, 1),
    ([5000 - 70 * n for n in range(64)], 64, 64, 28, 4),
]


@pytest.mark.parametrize(("lengths", "prefix", "page", "q_heads", "kv_heads"), SHARED)
def test_shared_prefix_of_infinite_values(lengths, prefix, page, q_heads, kv_heads):
    b = spoil(Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=20, prefix=prefix).fill(600), 21)
    q = normal((len(lengths), q_heads, 128), 22, 1.5)
    check(shared(b, q), b, q)
    b.page_table[:, :prefix] = b.prefix_pages
    check(decode(b, q), b, q)
    if min(lengths) > 0:  # a row of length 0 brings no token that prefill could place
        check(prefill(b, q), b, q)


# ------------------------------------------------------------------------------- a request gone wrong

def milliseconds(call):
    call()
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    call()
    end.record()
    torch.cuda.synchronize()
    return begin.elapsed_time(end)


@pytest.mark.parametrize(("what", "most"), [("k", 2.0), ("q", 2.0), ("v", 40.0)])
@pytest.mark.parametrize(("new", "past"), [([6000] + [100] * 20, [0] + [300] * 20), ([300, 60, 1], [9000, 2000, 4000])])
def test_a_spoiled_request_does_not_hold_up_the_others(new, past, what, most):
    """One NaN at the first position of a sequence, in whole blocks and in runs: the others' bits stay, and so does the
    order of the call's time. NaN scores need no more work than others; a NaN value has the sequence's rows attended again
    with the products of single warps. (Key by key, one row of 6000 keys took milliseconds, and there are 96000.)"""
    n = new[0]
    b = Batch(new, past, 64, 8, seed=23).fill(700)
    q = normal((b.tokens, 16, 128), 24, 1.5)
    good = prefill(b, q)
    before = milliseconds(lambda: prefill(b, q))
    pages, rows = b.places(0, 1)
    if what == "q":
        q[:n, :, 0] = NAN
    else:
        getattr(b, what)[pages, :, rows, 0] = NAN
    out = prefill(b, q)
    assert torch.equal(out[n:], good[n:])
    lost = torch.isnan(out[:n].view(n, 16, 128))
    assert lost[:, :, 0].all() and (what == "v" or lost.all())
    if what == "v":
        assert torch.equal(lost.sum(-1), torch.ones_like(lost[:, :, 0], dtype=torch.int64))
    assert nat.device_error() == 0
    assert milliseconds(lambda: prefill(b, q)) < most * before


@pytest.mark.parametrize(("cu", "sequences"), [
    ([0, 60, 0, 60, 100], 4), ([0, 60, 50, 60, 100], 4), ([0, 60, 90, 30, 100], 4), ([0, 60, 2 ** 30, 30, 60], 4), ([0, 0, -60, 0, 60], 4),
    ([0, 60, 0, 60, 100], 40), ([0, 60, 90, 30, 100], 1100)])
def test_prefill_offsets_that_are_no_offsets(cu, sequences):
    """Offsets that do not ascend, over values that are not finite: the sequences before are served, the rows of the others
    are left as they are, and so is what lies around the output."""
    sound = next(s for s in range(4) if not 0 <= cu[s] <= cu[s + 1] <= 100)
    b = spoil(Batch([60] + [40] * (sequences - 1), [300] * sequences, 16, 2, seed=25).fill(800), 26)
    q = normal((100, 4, 128), 27, 1.5)
    b.cu = torch.tensor(cu + [100] * (sequences - 4), dtype=torch.int32, device=DEV)
    guarded = torch.full((100 + 64, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    out = guarded[32:132]
    for _ in range(3):
        ops.paged_prefill_attention(q, b.k, b.v, b.page_table, b.cu, b.lengths, out)
        assert nat.device_error() == 2
    assert (guarded[:32] == 7).all() and (guarded[132:] == 7).all()
    served = cu[sound] if sound else 0
    b.new, b.tokens = [cu[i + 1] - cu[i] for i in range(sound)], served
    if served:
        check(out, b, q[:served])
    assert (out[served:] == 7).all()
