"""The operators over a paged cache against their definitions in 64 bits.

Tolerances, from the arithmetic. bf16 rounds by at most half a step, 2^-8 relative.
- append: q and k are computed in fp32 and rounded once: 2^-8 |y|, plus the fp32 chain (a sum of 128 squares, a root,
  three products, a sum), under 2^-18 of the two products' magnitudes. v is copied: equal.
- attention: the output is rounded once, 2^-8 |o|; the softmax weights may be rounded to bf16 before they meet v, which
  moves o by at most 2^-8 A, A = sum p |v| / sum p; a score in fp32 is off by at most 128 * 2^-24 sum |q_i k_i| / sqrt(128),
  under 2^-12 for these inputs, and moves o by at most twice that times A: 2^-11 A, the approximation of exp with it.
Unused rows of pages, and pages no sequence has, hold NaN: nothing of them may reach an output.
"""

import math

import pytest
import torch

from ipe_b200 import _native as nat
from ipe_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8
EPS = 1e-6
NAN = float("nan")


class Batch:
    """Sequences with new tokens on top of `past` positions, their pages dealt out in no order, the cache NaN."""

    def __init__(self, new, past, page, kv_heads, seed, spare=3, prefix=0, pages_to_spare_first=0):
        self.new, self.length = list(new), [n + p for n, p in zip(new, past)]
        self.page, self.kv_heads, self.prefix = page, kv_heads, prefix
        g = torch.Generator().manual_seed(seed)
        counts = [max(0, -(-n // page) - prefix) for n in self.length]
        total = prefix + sum(counts) + spare
        order = torch.randperm(total, generator=g).tolist()
        order = [p + pages_to_spare_first for p in order]
        self.prefix_ids = order[:prefix]
        at, table, width = prefix, [], prefix + max(counts, default=0) + 1
        for c in counts:
            table.append(([-7] * prefix + order[at:at + c] + [10 ** 9] * width)[:width])
            at += c
        self.table = table
        shape = (total + pages_to_spare_first, kv_heads, page, 128)
        self.k = torch.full(shape, NAN, dtype=torch.bfloat16, device=DEV)
        self.v = torch.full(shape, NAN, dtype=torch.bfloat16, device=DEV)
        as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        self.page_table = as_int(table).reshape(len(table), width)
        self.lengths, self.prefix_pages = as_int(self.length), as_int(self.prefix_ids)
        self.cu = as_int([sum(self.new[:s]) for s in range(len(self.new) + 1)])
        self.tokens = sum(self.new)

    def places(self, s, count=None, start=0):
        """(page, row) index tensors of positions start .. of sequence s."""
        positions = torch.arange(start, self.length[s] if count is None else count)
        ids = torch.tensor((self.prefix_ids + self.table[s][self.prefix:]) or [0])
        return ids[positions // self.page].to(DEV), (positions % self.page).to(DEV)

    def fill(self, seed, scale=1.0):
        """Every position of every sequence gets keys and values (the shared ones once)."""
        for s in range(len(self.new)):
            pages, rows = self.places(s)
            self.k[pages, :, rows] = normal((len(rows), self.kv_heads, 128), seed + 2 * s, scale)
            self.v[pages, :, rows] = normal((len(rows), self.kv_heads, 128), seed + 2 * s + 1)
        return self

    def keys(self, s, kv_head, count):
        pages, rows = self.places(s, count)
        return self.k[pages, kv_head, rows].double(), self.v[pages, kv_head, rows].double()


def normal(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def attend(batch, q):
    """(o, A) in 64 bits [tokens, Hq * 128] by the definition, one sequence and head at a time."""
    heads = q.shape[1]
    o = torch.zeros(batch.tokens, heads, 128, dtype=torch.float64, device=DEV)
    a = torch.zeros_like(o)
    at = 0
    for s, n in enumerate(batch.new):
        total = batch.length[s]
        for h in range(heads):
            if total == 0 or n == 0:
                continue
            k, v = batch.keys(s, h // (heads // batch.kv_heads), total)
            score = q[at:at + n, h].double() @ k.T / math.sqrt(128)
            hidden = torch.arange(total, device=DEV) > (total - n + torch.arange(n, device=DEV))[:, None]
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            # values behind a row's last key do not belong to it, whatever they are
            for x, y in ((o, v), (a, v.abs())):
                finite = torch.isfinite(y)
                part = p @ torch.where(finite, y, 0.0)
                bad = (~hidden).double() @ (~finite).double()
                x[at:at + n, h] = torch.where(bad > 0, NAN, part)
        at += n
    return o.view(batch.tokens, -1), a.view(batch.tokens, -1)


def check(out, batch, q):
    o, a = attend(batch, q)
    got = out[:batch.tokens].double()
    lost = torch.isnan(o)
    assert torch.equal(lost, ~torch.isfinite(got))
    over = ((got - o).abs() - (HALF * o.abs() + (HALF + 2.0 ** -11) * a))[~lost]
    assert over.numel() == 0 or float(over.max()) <= 0
    assert nat.device_error() == 0


def decode(batch, q):
    out = torch.full((len(batch.new), q.shape[1] * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    return ops.paged_decode_attention(q, batch.k, batch.v, batch.page_table, batch.lengths, out)


def prefill(batch, q):
    out = torch.full((q.shape[0], q.shape[1] * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    return ops.paged_prefill_attention(q, batch.k, batch.v, batch.page_table, batch.cu, batch.lengths, out)


def shared(batch, q):
    out = torch.full((q.shape[0], q.shape[1] * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    return ops.shared_prefix_attention(q, batch.k, batch.v, batch.prefix_pages, batch.page_table, batch.lengths, out)


# ------------------------------------------------------------------------------------------ append

def append_reference(batch, qkv, q_heads, q_norm, k_norm, cos, sin):
    """(y, magnitude) in 64 bits of every new token's q and k heads [tokens, Hq + Hkv, 128]."""
    heads = q_heads + batch.kv_heads
    x = qkv[:batch.tokens].double().view(batch.tokens, -1, 128)[:, :heads]
    weight = torch.cat((q_norm.double().expand(q_heads, 128), k_norm.double().expand(batch.kv_heads, 128)))
    y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight
    pos = torch.cat([torch.arange(t - n, t) for n, t in zip(batch.new, batch.length)]).to(DEV)
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    turned = torch.cat((-y[..., 64:], y[..., :64]), -1)
    return y * c + turned * s, (y * c).abs() + (turned * s).abs()


@pytest.mark.parametrize(("new", "past", "page", "q_heads", "kv_heads", "table", "behind"), [
    ([1], [0], 16, 16, 8, torch.bfloat16, 0),
    ([1, 1, 1], [0, 15, 16], 16, 4, 1, torch.float32, 0),
    ([3, 0, 40, 1, 0], [14, 9, 0, 700, 0], 16, 16, 8, torch.bfloat16, 5),
    ([64, 65, 1], [0, 63, 127], 64, 40, 8, torch.float32, 1),
    ([129], [1], 128, 6, 2, torch.bfloat16, 17),
    ([2] * 70, list(range(70)), 32, 8, 1, torch.bfloat16, 0),
    ([7, 300], [33, 0], 32, 2, 2, torch.float32, 130),
])
def test_append(new, past, page, q_heads, kv_heads, table, behind):
    b = Batch(new, past, page, kv_heads, seed=1)
    rows = b.tokens + behind
    qkv = normal((rows, (q_heads + 2 * kv_heads) * 128), 2)
    qkv[0] *= 1e-3  # a row whose epsilon counts
    qkv[b.tokens:] = NAN
    q_norm, k_norm = 1 + normal((128,), 3, 0.2), 1 + normal((128,), 4, 0.2)
    angle = torch.arange(max(b.length) or 1, device=DEV)[:, None] * (1e6 ** (-torch.arange(64, device=DEV) / 64.0)).repeat(2)
    cos, sin = angle.cos().to(table), angle.sin().to(table)
    q_out = torch.full((rows, q_heads, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_qk_norm_rope_append(qkv, q_norm, k_norm, cos, sin, b.cu, b.lengths, b.page_table, EPS, q_out, b.k, b.v)
    assert nat.device_error() == 0
    y, size = append_reference(b, qkv, q_heads, q_norm, k_norm, cos, sin)
    limit = HALF * y.abs() + 2.0 ** -18 * size
    assert ((q_out[:b.tokens].double() - y[:, :q_heads]).abs() <= limit[:, :q_heads]).all()
    assert (q_out[b.tokens:] == 7).all()
    v = qkv.view(rows, -1, 128)[:, q_heads + kv_heads:]
    at, written = 0, torch.zeros(b.k.shape[0], page, dtype=torch.bool, device=DEV)
    for s, n in enumerate(new):
        pages, place = b.places(s, start=past[s])
        assert ((b.k[pages, :, place].double() - y[at:at + n, q_heads:]).abs() <= limit[at:at + n, q_heads:]).all()
        assert torch.equal(b.v[pages, :, place], v[at:at + n])
        written[pages, place] = True
        at += n
    for cache in (b.k, b.v):
        assert torch.isnan(cache.transpose(1, 2)[~written]).all(), "a row that no token has was written"


def test_append_without_a_place():
    """Tokens that have no page or no position are skipped and reported; the others are served."""
    b = Batch([2, 1, 1, 1], [0, 4, 5, 6], 16, 2, seed=5)
    qkv, w = normal((5, 8 * 128), 6), torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cos, sin = torch.ones(6, 128, device=DEV), torch.zeros(6, 128, device=DEV)
    for sequence, column, value, code in ((1, "page_table", b.k.shape[0], 5), (1, "page_table", -1, 5),
                                          (2, "lengths", 40, 2), (2, "lengths", -3, 2), (0, "lengths", 1, 2)):
        b.k.fill_(NAN)
        broken = {"page_table": b.page_table.clone(), "lengths": b.lengths.clone()}
        broken[column].view(len(b.new), -1)[sequence, 0] = value
        q_out = torch.full((5, 4, 128), 7.0, dtype=torch.bfloat16, device=DEV)
        lengths = broken["lengths"].clone()
        lengths[3] = 6  # position 5: inside the tables
        ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, b.cu, lengths, broken["page_table"], EPS, q_out, b.k, b.v)
        assert nat.device_error() == code
        written = (~torch.isnan(b.k[:, 0, :, 0])).sum()
        assert int(written) == 4
    ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, b.cu, b.lengths, b.page_table, EPS, q_out, b.k, b.v)
    assert nat.device_error() == 2  # sequence 3's position 6 is past the tables of 6 rows


# ------------------------------------------------------------------------------------------ decode

DECODE = [
    ([1], 16, 16, 8),
    ([640], 16, 16, 8),
    ([0, 1, 15, 16, 17, 31, 32, 33], 16, 4, 2),
    ([127, 128, 129, 0, 255, 256, 257], 32, 3, 1),
    ([5000, 1, 0, 300], 64, 40, 8),
    ([1000, 77], 128, 28, 4),
    ([64, 65, 63], 64, 12, 2),
    ([2049], 128, 8, 1),
    ([9] * 200, 16, 2, 2),
    (list(range(300, 360)), 32, 32, 8),
    ([33000, 5, 12000], 16, 7, 1),
]


@pytest.mark.parametrize(("lengths", "page", "q_heads", "kv_heads"), DECODE)
def test_decode(lengths, page, q_heads, kv_heads):
    b = Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=7).fill(100)
    q = normal((len(lengths), q_heads, 128), 8, 1.5)
    out = decode(b, q)
    check(out, b, q)
    assert torch.equal(out, decode(b, q))  # the same bits again
    assert (out[b.lengths == 0] == 0).all()


def test_decode_large_and_small_scores():
    """Scores of several hundred, where a softmax without its maximum overflows, and rows where one key has it all."""
    b = Batch([1] * 3, [300, 40, 1000], 16, 2, seed=9).fill(200, scale=6.0)
    q = normal((3, 4, 128), 10, 6.0)
    o, _ = attend(b, q)
    # scores up to ~500: off by up to 128 * 2^-24 * 500 * 4, so p by up to 1.6 %
    assert ((decode(b, q).double() - o).abs() <= 0.016 * 2 * b.v[~torch.isnan(b.v)].abs().max().double() + HALF * o.abs()).all()
    assert nat.device_error() == 0


def test_decode_reports_what_it_cannot_read():
    b = Batch([1] * 3, [40, 50, 60], 16, 2, seed=11).fill(300)
    q = normal((3, 4, 128), 12)
    good = decode(b, q)
    for column, value, code in (("page_table", b.k.shape[0], 5), ("page_table", -2, 5), ("lengths", 16 * 99, 2), ("lengths", -1, 2)):
        keep = getattr(b, column).clone()
        getattr(b, column).view(3, -1)[1, 0] = value
        out = decode(b, q)
        assert nat.device_error() == code
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
        setattr(b, column, keep)


# ----------------------------------------------------------------------------------------- prefill

PREFILL = [
    ([1], [0], 16, 16, 8, 0),
    ([1, 2, 3], [0, 0, 5], 16, 4, 2, 2),
    ([128], [0], 16, 16, 8, 0),
    ([127, 129, 1, 0, 64], [0, 0, 0, 50, 0], 32, 16, 8, 3),
    ([300, 17, 1], [0, 1000, 4000], 64, 8, 2, 40),
    ([257], [0], 128, 5, 1, 0),
    ([100, 100], [129, 31], 16, 6, 2, 0),
    ([65, 1, 200], [63, 128, 700], 128, 28, 4, 1),
    ([1000], [0], 64, 16, 8, 0),
    ([513], [2000], 16, 8, 1, 9),
    ([4] * 60, [n * 7 for n in range(60)], 16, 32, 8, 0),
    ([40], [30000], 32, 16, 8, 0),
    ([1500, 3], [0, 11], 16, 2, 2, 0),
    ([(37 * n) % 211 for n in range(40)], [(91 * n) % 517 for n in range(40)], 16, 24, 8, 2),  # whole blocks, many per CTA
    ([700, 1, 900, 40], [0, 3000, 100, 1], 128, 64, 8, 0),
    ([n % 3 for n in range(1100)], [n % 5 for n in range(1100)], 16, 8, 8, 0),  # more sequences than are listed at once
]


@pytest.mark.parametrize(("new", "past", "page", "q_heads", "kv_heads", "behind"), PREFILL)
def test_prefill(new, past, page, q_heads, kv_heads, behind):
    b = Batch(new, past, page, kv_heads, seed=13).fill(400)
    q = normal((b.tokens + behind, q_heads, 128), 14, 1.5)
    q[b.tokens:] = NAN
    out = prefill(b, q)
    check(out, b, q)
    assert (out[b.tokens:] == 7).all()
    again = prefill(b, q)
    assert torch.equal(out, again)


def test_prefill_more_tokens_than_positions():
    """A sequence that brings more tokens than its length counts: reported; the others are served."""
    b = Batch([5, 4], [20, 6], 16, 2, seed=15).fill(500)
    q = normal((9, 4, 128), 16)
    good = prefill(b, q)
    b.lengths[0] = 3
    out = prefill(b, q)
    assert nat.device_error() == 2
    assert torch.equal(out[5:], good[5:])
    assert (out[:2] == 0).all()  # no position at all


def test_prefill_offsets_that_are_no_offsets():
    """cu_tokens that decrease or pass the rows: nothing outside the buffers is touched."""
    b = Batch([5, 4], [20, 6], 16, 2, seed=17).fill(600)
    q = normal((9, 4, 128), 18)
    for cu in ([0, 9000, 9], [0, 5, 2 ** 31 - 1], [7, 3, 1], [-5, -3, -1], [4, 4, 4]):
        b.cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
        guarded = torch.full((9 + 64, 512), 7.0, dtype=torch.bfloat16, device=DEV)
        ops.paged_prefill_attention(q, b.k, b.v, b.page_table, b.cu, b.lengths, guarded[32:41])
        nat.device_error()
        assert (guarded[:32] == 7).all() and (guarded[41:] == 7).all()


@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
def test_later_positions_do_not_reach_earlier_rows(bad):
    """Keys and values of a sequence's own later tokens, whatever they hold, are not seen by the rows before them."""
    b = Batch([200], [30], 16, 2, seed=19).fill(700)
    q = normal((200, 4, 128), 20)
    o, a = attend(b, q)
    pages, rows = b.places(0, start=150)
    b.v[pages, :, rows] = bad
    b.k[pages, 1:, rows] = bad
    out = prefill(b, q)
    first = 150 - 30
    assert ((out.double() - o).abs() <= HALF * o.abs() + (HALF + 2.0 ** -11) * a)[:first].all()
    assert nat.device_error() == 0


@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_later_positions_beside_many_other_sequences(bad):
    """The same where blocks stay whole, and every other sequence as it was."""
    new = [150] * 40
    b = Batch(new, [20] * 40, 16, 8, seed=19).fill(700)
    q = normal((b.tokens, 8, 128), 20)
    o, a = attend(b, q)
    for s in (0, 17):
        pages, rows = b.places(s, start=100)
        b.v[pages, :, rows] = bad
    out = prefill(b, q)
    close = ((out.double() - o).abs() <= HALF * o.abs() + (HALF + 2.0 ** -11) * a).all(-1).view(40, 150)
    sees = torch.zeros(40, 150, dtype=torch.bool, device=DEV)
    sees[0, 80:] = sees[17, 80:] = True
    assert torch.equal(close, ~sees)
    assert not torch.isfinite(out.view(40, 150, -1)[sees]).any()
    assert nat.device_error() == 0


# ------------------------------------------------------------------------------------------ shared

SHARED = [
    ([33, 40, 64], 2, 16, 16, 8),
    ([32, 31, 1, 0, 33], 2, 16, 4, 2),
    ([200], 3, 64, 8, 1),
    ([700 + 3 * n for n in range(20)], 40, 16, 16, 8),
    ([1300 + n % 50 for n in range(130)], 20, 64, 40, 8),
    ([513 + 128 * n for n in range(9)], 4, 128, 3, 1),
    ([5, 17, 0], 0, 16, 4, 2),
    ([8200, 8193], 64, 128, 12, 2),
    ([2048 + 13 * n for n in range(64)], 64, 32, 28, 4),
    ([1024] * 33, 32, 32, 32, 8),
    ([33 + n % 40 for n in range(700)], 2, 16, 64, 8),  # more blocks of rows than CTAs
    ([2600 + n for n in range(5)], 81, 32, 14, 2),
]


@pytest.mark.parametrize(("lengths", "prefix", "page", "q_heads", "kv_heads"), SHARED)
def test_shared_prefix(lengths, prefix, page, q_heads, kv_heads):
    b = Batch([1] * len(lengths), [n - 1 for n in lengths], page, kv_heads, seed=21, prefix=prefix).fill(800)
    q = normal((len(lengths), q_heads, 128), 22, 1.5)
    out = shared(b, q)
    check(out, b, q)
    assert torch.equal(out, shared(b, q))
    assert (out[b.lengths == 0] == 0).all()


@pytest.mark.parametrize(("q_heads", "kv_heads"), [(4, 2), (3, 1)])
def test_shared_prefix_of_more_sequences_than_are_listed(q_heads, kv_heads):
    b = Batch([1] * 1100, [n % 90 for n in range(1100)], 32, kv_heads, seed=29, prefix=2).fill(970)
    q = normal((1100, q_heads, 128), 30, 1.5)
    check(shared(b, q), b, q)


@pytest.mark.parametrize("bad", [NAN, float("inf"), torch.finfo(torch.bfloat16).min])
def test_shared_keys_behind_a_rows_end(bad):
    """A sequence that ends inside the prefix sees nothing of the prefix's later keys, whatever they hold."""
    b = Batch([1] * 4, [39, 70, 150, 129], 16, 2, seed=27, prefix=12).fill(950)
    q = normal((4, 8, 128), 28, 1.5)
    o, a = attend(b, q)
    pages, rows = b.places(0, count=192, start=151)
    b.v[pages, :, rows] = bad
    b.k[pages, 1:, rows] = bad
    out = shared(b, q)
    assert ((out.double() - o).abs() <= HALF * o.abs() + (HALF + 2.0 ** -11) * a).all()
    assert nat.device_error() == 0


def test_shared_prefix_is_paged_decode_on_whole_tables():
    b = Batch([1] * 6, [900 + 60 * n for n in range(6)], 32, 2, seed=23, prefix=20).fill(900)
    q = normal((6, 8, 128), 24)
    out = shared(b, q)
    b.page_table[:, :20] = b.prefix_pages
    whole = decode(b, q)
    o, a = attend(b, q)
    assert ((out.double() - whole.double()).abs() <= 2 * (HALF * o.abs() + (HALF + 2.0 ** -11) * a)).all()


def test_shared_prefix_reports_what_it_cannot_read():
    b = Batch([1] * 3, [40, 50, 60], 16, 2, seed=25, prefix=2).fill(1000)
    q = normal((3, 4, 128), 26)
    shared(b, q)
    assert nat.device_error() == 0
    b.prefix_pages[1] = b.k.shape[0]
    shared(b, q)
    assert nat.device_error() == 5
    b.prefix_pages[1] = b.prefix_ids[1]
    good = shared(b, q)
    b.page_table[1, 2] = -1
    out = shared(b, q)
    assert nat.device_error() == 5
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])


# ---------------------------------------------------------------------------------------- together

def test_prompts_in_pieces_then_answers():
    """A server's steps: prompts arrive in pieces beside running requests, then every request decodes; each step appends
    and attends, and every output is checked from what the cache holds."""
    q_heads, kv_heads, page = 8, 4, 16
    final = [75, 140, 33]
    b = Batch(final, [0, 0, 0], page, kv_heads, seed=27)
    w = 1 + normal((128,), 28, 0.1)
    angle = torch.arange(160, device=DEV)[:, None] * (1e6 ** (-torch.arange(64, device=DEV) / 64.0)).repeat(2)
    cos, sin = angle.cos().bfloat16(), angle.sin().bfloat16()
    length = [0, 0, 0]
    for step, new in enumerate([[60, 0, 0], [10, 100, 0], [1, 35, 30], [1, 1, 1], [1, 1, 1]]):
        length = [n + m for n, m in zip(length, new)]
        b.new, b.length, b.tokens = new, length, sum(new)
        b.cu = torch.tensor([sum(new[:s]) for s in range(4)], dtype=torch.int32, device=DEV)
        b.lengths = torch.tensor(length, dtype=torch.int32, device=DEV)
        qkv = normal((b.tokens, (q_heads + 2 * kv_heads) * 128), 30 + step)
        q = torch.empty(b.tokens, q_heads, 128, dtype=torch.bfloat16, device=DEV)
        ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, b.cu, b.lengths, b.page_table, EPS, q, b.k, b.v)
        y, size = append_reference(b, qkv, q_heads, w, w, cos, sin)
        assert ((q.double() - y[:, :q_heads]).abs() <= HALF * y[:, :q_heads].abs() + 2.0 ** -18 * size[:, :q_heads]).all()
        check(prefill(b, q), b, q)
        if set(new) == {1}:
            check(decode(b, q), b, q)
    assert nat.device_error() == 0


def test_replays_with_other_lengths_and_tables():
    """One captured decode step (append, decode, shared, prefill of the same rows) serves growing and idle rows."""
    b = Batch([1] * 4, [200, 90, 300, 150], 16, 2, seed=40, prefix=3).fill(1100)
    whole = b.page_table.clone()
    whole[:, :3] = b.prefix_pages
    q_heads = 6
    qkv = normal((4, (q_heads + 4) * 128), 41)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cos, sin = torch.ones(400, 128, device=DEV), torch.zeros(400, 128, device=DEV)
    q = torch.zeros(4, q_heads, 128, dtype=torch.bfloat16, device=DEV)
    outs = [torch.zeros(4, q_heads * 128, dtype=torch.bfloat16, device=DEV) for _ in range(3)]

    def step():
        ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, b.cu, b.lengths, whole, EPS, q, b.k, b.v)
        ops.paged_decode_attention(q, b.k, b.v, whole, b.lengths, outs[0])
        ops.shared_prefix_attention(q, b.k, b.v, b.prefix_pages, b.page_table, b.lengths, outs[1])
        ops.paged_prefill_attention(q, b.k, b.v, whole, b.cu, b.lengths, outs[2])

    step()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    with torch.cuda.graph(other):  # a second captured step beside the first
        step()
    for lengths in ([201, 91, 301, 151], [60, 49, 300, 52], [100, 50, 64, 65]):
        b.length = lengths
        b.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        qkv.copy_(normal(qkv.shape, sum(lengths)))
        graph.replay()
        other.replay()
        for out in outs:
            check(out, b, q)


def test_a_captured_step_behind_copies_and_fills():
    """The operators' kernels start early behind other kernels; behind copies and fills, captured too, they read what
    those wrote."""
    b = Batch([1] * 3, [100, 60, 200], 16, 2, seed=42).fill(1150)
    q_new = normal((3, 4, 128), 43)
    q, out = torch.zeros_like(q_new), torch.zeros(3, 512, dtype=torch.bfloat16, device=DEV)
    lengths_new = b.lengths.clone()

    def step():
        b.lengths.zero_()
        ops.paged_decode_attention(q, b.k, b.v, b.page_table, b.lengths, out)
        b.lengths.copy_(lengths_new)
        q.copy_(q_new)
        ops.paged_decode_attention(q, b.k, b.v, b.page_table, b.lengths, out)
        out_first.copy_(out)
        ops.paged_prefill_attention(q, b.k, b.v, b.page_table, b.cu, b.lengths, out)

    out_first = torch.zeros_like(out)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for round_ in range(3):
        q_new.copy_(normal(q_new.shape, 44 + round_))
        graph.replay()
        torch.cuda.synchronize()
        check(out_first, b, q_new)
        check(out, b, q_new)


def test_calls_on_two_streams_at_once():
    batches = [Batch([1] * 5, [700 + 90 * n + s for n in range(5)], 32, 2, seed=50 + s, prefix=10).fill(1200 + 50 * s) for s in range(2)]
    queries = [normal((5, 8, 128), 60 + s) for s in range(2)]
    for b in batches:
        b.whole = b.page_table.clone()
        b.whole[:, :10] = b.prefix_pages
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                b, q = batches[i], queries[i]
                o = [torch.empty(5, 8 * 128, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
                ops.paged_decode_attention(q, b.k, b.v, b.whole, b.lengths, o[0])
                ops.shared_prefix_attention(q, b.k, b.v, b.prefix_pages, b.page_table, b.lengths, o[1])
                ops.paged_prefill_attention(q, b.k, b.v, b.whole, b.cu, b.lengths, o[2])
                outs[i].append(o)
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            for out in o:
                check(out, batches[i], queries[i])


def test_pages_behind_the_first_four_billion_bytes():
    """A cache whose rows lie past 2^31 elements and 2^32 bytes."""
    ahead = 2 ** 31 // (8 * 128 * 128) + 40
    b = Batch([3, 1], [200, 400], 128, 8, seed=70, pages_to_spare_first=ahead).fill(1300)
    assert b.k.numel() > 2 ** 31
    q = normal((4, 16, 128), 71)
    check(prefill(b, q), b, q)
    b.new, b.tokens = [1, 1], 2
    check(decode(b, q[:2].contiguous()), b, q[:2])
    qkv = normal((2, 32 * 128), 72)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cos, sin = torch.ones(500, 128, device=DEV), torch.zeros(500, 128, device=DEV)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    ops.paged_qk_norm_rope_append(qkv, w, w, cos, sin, cu, b.lengths, b.page_table, EPS, q[:2], b.k, b.v)
    for s in range(2):
        pages, rows = b.places(s, start=b.length[s] - 1)
        assert torch.equal(b.v[pages, :, rows][0], qkv[s].view(32, 128)[24:])
    assert nat.device_error() == 0


def test_nothing_to_do():
    b = Batch([1], [0], 16, 2, seed=80)
    none = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(0, 512, dtype=torch.bfloat16, device=DEV)
    ops.paged_prefill_attention(none, b.k, b.v, b.page_table, b.cu * 0, b.lengths, out)
    empty = b.page_table[:0], b.lengths[:0]
    ops.paged_decode_attention(none, b.k, b.v, *empty, out)
    ops.shared_prefix_attention(none, b.k, b.v, b.prefix_pages, *empty, out)
    assert nat.device_error() == 0


def test_the_registered_operators():
    b = Batch([1] * 2, [40, 50], 16, 2, seed=90, prefix=1).fill(1400)
    q = normal((2, 4, 128), 91)
    out = torch.empty(2, 512, dtype=torch.bfloat16, device=DEV)
    torch.ops.ipe_b200.shared_prefix_attention(q, b.k, b.v, b.prefix_pages, b.page_table, b.lengths, out)
    check(out, b, q)
    b.page_table[:, :1] = b.prefix_pages
    torch.ops.ipe_b200.paged_decode_attention(q, b.k, b.v, b.page_table, b.lengths, out.zero_())
    check(out, b, q)
    torch.ops.ipe_b200.paged_prefill_attention(q, b.k, b.v, b.page_table, b.cu, b.lengths, out.zero_())
    check(out, b, q)
    qkv, w = normal((2, 8 * 128), 92), torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cos, sin = torch.ones(60, 128, device=DEV), torch.zeros(60, 128, device=DEV)
    torch.ops.ipe_b200.paged_qk_norm_rope_append(qkv, w, w, cos, sin, b.cu, b.lengths, b.page_table, EPS, q, b.k, b.v)
    pages, rows = b.places(0, start=40)
    assert torch.equal(b.v[pages, :, rows][0], qkv[0].view(8, 128)[6:])


def test_subclasses_of_tensor_and_whole_numbers():
    """What the extension module leaves to the Python checks gives the same bits."""
    class Other(torch.Tensor):
        pass

    b = Batch([3, 1], [40, 50], 16, 2, seed=97, prefix=1).fill(1500)
    qkv, w = normal((4, 8 * 128), 98), torch.ones(128, dtype=torch.bfloat16, device=DEV)
    cos, sin = normal((60, 128), 99, dtype=torch.float32), normal((60, 128), 100, dtype=torch.float32)
    b.page_table[:, :1] = b.prefix_pages
    rows = []
    for eps, change in ((1.0, lambda t: t), (1, lambda t: t), (1.0, lambda t: t.as_subclass(Other)),
                        (1.0, lambda t: torch.nn.Parameter(t, requires_grad=False))):
        q = torch.empty(4, 4, 128, dtype=torch.bfloat16, device=DEV)
        k, v, table, lengths = change(b.k.clone()), change(b.v.clone()), change(b.page_table), change(b.lengths)
        ops.paged_qk_norm_rope_append(change(qkv), w, w, cos, sin, b.cu, lengths, table, eps, change(q), k, v)
        outs = [torch.empty(4, 512, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
        ops.paged_prefill_attention(change(q), k, v, table, b.cu, lengths, outs[0])
        ops.paged_decode_attention(q[2:].contiguous(), k, v, table, lengths, change(outs[1][:2]))
        ops.shared_prefix_attention(change(q[2:].contiguous()), k, v, b.prefix_pages, table, lengths, outs[2][:2])
        rows.append([q, k, v, outs[0], outs[1][:2], outs[2][:2]])
    for other in rows[1:]:
        for x, y in zip(rows[0], other):
            assert torch.equal(torch.nan_to_num(x.as_subclass(torch.Tensor).detach()), torch.nan_to_num(y.as_subclass(torch.Tensor).detach()))
    assert nat.device_error() == 0


def test_refusals_of_the_python_functions():
    b = Batch([1] * 2, [40, 50], 16, 2, seed=95)
    q = normal((2, 4, 128), 96)
    out = torch.empty(2, 512, dtype=torch.bfloat16, device=DEV)
    good = dict(q=q, k_pages=b.k, v_pages=b.v, page_table=b.page_table, lengths=b.lengths, out=out)
    for change in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[:, :, :64].contiguous()), dict(q=q[:, :3].contiguous()),
                   dict(q=normal((2, 8, 128), 1)[:, ::2]), dict(k_pages=b.k[:1]), dict(v_pages=b.v.half()),
                   dict(k_pages=b.k.transpose(1, 2)), dict(page_table=b.page_table.long()), dict(page_table=b.page_table[:, 0]),
                   dict(page_table=b.page_table[:, :2]), dict(lengths=b.lengths[:1]), dict(lengths=b.lengths.cpu()),
                   dict(out=out[:, :256]), dict(out=out.float())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_decode_attention(**{**good, **change})
    for cu in (b.cu[:2], b.cu.long(), b.cu.cpu()):
        with pytest.raises(ValueError):
            ops.paged_prefill_attention(q, b.k, b.v, b.page_table, cu, b.lengths, out)
    for prefix in (b.cu.view(1, 3), torch.zeros(99, dtype=torch.int32, device=DEV), b.cu.long()):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(q, b.k, b.v, prefix, b.page_table, b.lengths, out)
    wide = normal((2, 2, 16, 128), 2)[:, :, :, :].repeat(1, 1, 2, 1)[:, :, :24].contiguous()
    with pytest.raises(RuntimeError, match="page_size"):
        ops.paged_decode_attention(q, wide, wide, b.page_table, b.lengths, out)
    assert nat.device_error() == 0
