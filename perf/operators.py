"""The paged-cache operators of `ipe_b200.ops`, as calls to measure: the append of rotated keys and values, the two
attentions that read the pages, and the decode attention of a batch that shares its prompt's beginning.

A cache is two tensors of pages [pages, KV heads, page size, 128]; sequence s keeps its position p in page
page_table[s, p // page size], row p % page size. A batch of new tokens is ragged: sequence s brings rows
cu_tokens[s] .. cu_tokens[s + 1] - 1, the last ones of its lengths[s] positions.

`listed` names the cases, `draw` makes more of the same ranges, `prepare` makes a case's inputs on the GPU, `run` is one
call (the plain form in elementary torch operations, or the framework's operator where `own` is true), `exact` the
definition in 64 bits, `work` the bytes and operations that the call cannot do without.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

HEAD = 128
EPS = 1e-6
THETA = 1e6
SCALE = HEAD ** -0.5


# ------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step's append for 16 running requests
        dict(name="append-decode-16", op="append", q_heads=16, kv_heads=8, page=16, sequences=16, new_low=1, new_high=1,
             past_low=40, past_high=1000, behind=0, table="bf16"),
        # a step that mixes running requests with pieces of new prompts, in a buffer of fixed size (rows behind the last)
        dict(name="append-mixed", op="append", q_heads=32, kv_heads=8, page=32, sequences=24, new_low=1, new_high=509,
             past_low=1, past_high=4000, behind=61, table="fp32"),
        # whole prompts, long and short
        dict(name="append-prompts", op="append", q_heads=16, kv_heads=8, page=64, sequences=12, new_low=33, new_high=8192,
             past_low=0, past_high=0, behind=0, table="bf16"),
        # one request in the middle of its answer, the latency case
        dict(name="decode-1", op="decode", q_heads=16, kv_heads=8, page=16, sequences=1, low=640, high=640, idle=0),
        # 16 requests, one of them far longer than the rest, in small pages
        dict(name="decode-16-uneven", op="decode", q_heads=16, kv_heads=8, page=16, sequences=16, low=90, high=30001, idle=0),
        # a full server: 64 requests of a model with 5 query heads to a KV head, two rows of the captured batch unused
        dict(name="decode-64", op="decode", q_heads=40, kv_heads=8, page=64, sequences=64, low=700, high=12289, idle=2),
        # one prompt of the benchmark's length
        dict(name="prefill-512", op="prefill", q_heads=16, kv_heads=8, page=16, sequences=1, new_low=512, new_high=512,
             past_low=0, past_high=0, behind=0),
        # prompts of uneven lengths together
        dict(name="prefill-ragged", op="prefill", q_heads=32, kv_heads=8, page=32, sequences=9, new_low=17, new_high=2500,
             past_low=0, past_high=0, behind=29),
        # pieces of two prompts on top of long contexts
        dict(name="prefill-on-context", op="prefill", q_heads=16, kv_heads=8, page=64, sequences=2, new_low=64, new_high=200,
             past_low=9000, past_high=20000, behind=0),
        # one long prompt
        dict(name="prefill-8192", op="prefill", q_heads=16, kv_heads=8, page=128, sequences=1, new_low=8192, new_high=8192,
             past_low=0, past_high=0, behind=0),
        # 12 answers to one question
        dict(name="shared-12", op="shared", q_heads=16, kv_heads=8, page=16, sequences=12, prefix=1504, low=3, high=250),
        # a server whose requests all begin with one long instruction
        dict(name="shared-160", op="shared", q_heads=32, kv_heads=8, page=64, sequences=160, prefix=16384, low=5, high=1100),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1)) - 0.5 / high))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "shared"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    case = dict(op=op, q_heads=kv_heads * rng.choice([1, 2, 2, 3, 4, 5, 8]), kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]))
    if op == "append":
        sequences = _log_int(rng, 1, 64)
        most = max(1, min(8192, 24000 * 32 // (case["q_heads"] + 2 * kv_heads) // sequences))
        case.update(sequences=sequences, new_low=1, new_high=_log_int(rng, 1, most), past_low=rng.choice([0, 5]),
                    past_high=_log_int(rng, 5, 4000), behind=rng.choice([0, 0, rng.randint(1, 70)]),
                    table=rng.choice(["bf16", "fp32"]))
    elif op == "decode":
        sequences = _log_int(rng, 1, 64)
        high = _log_int(rng, 4, min(30000, 250_000 // sequences))
        case.update(sequences=sequences, low=rng.randint(1, high), high=high, idle=rng.choice([0, 0, 1, 3]))
    elif op == "prefill":
        sequences = _log_int(rng, 1, 10)
        high = _log_int(rng, 2, min(8192, 14000 // sequences, int(2500 * (128 / case["q_heads"]) ** 0.5)))
        past = _log_int(rng, 2, 8000) if high < 600 else 0
        case.update(sequences=sequences, new_low=rng.randint(1, high), new_high=high, past_low=past // 3, past_high=past,
                    behind=rng.choice([0, 0, rng.randint(1, 70)]))
    else:
        sequences = _log_int(rng, 2, 160)
        case.update(sequences=sequences, prefix=case["page"] * _log_int(rng, 1, 12000 // case["page"]), low=1,
                    high=_log_int(rng, 1, 1000))
    return case


def _numbers(case, low, high, salt):
    """One number for each sequence, log-uniform in [low, high], the first of them `high`."""
    rng = random.Random(f"{case['sequences']} {low} {high} {salt}")
    rest = [low if high <= low else low - 1 + _log_int(rng, 1, high - low + 1) for _ in range(case["sequences"] - 1)]
    return [high, *rest]


def _sizes(case):
    """(new tokens of each sequence, its length with them)."""
    if case["op"] in ("append", "prefill"):
        new = _numbers(case, case["new_low"], case["new_high"], "new")
        past = _numbers(case, case["past_low"], case["past_high"], "past")
        past = past[len(past) // 2:] + past[:len(past) // 2]
        return new, [n + p for n, p in zip(new, past)]
    new = [1] * case["sequences"]
    if case["op"] == "decode":
        length = _numbers(case, case["low"], case["high"], "length")
        idle = min(case["idle"], len(length) - 1)
        return new, length[:len(length) - idle] + [0] * idle
    return new, [case["prefix"] + n for n in _numbers(case, case["low"], case["high"], "own")]


# ------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    hq, hkv, page, rows = case["q_heads"], case["kv_heads"], case["page"], case["sequences"]
    new, length = _sizes(case)
    prefix = case.get("prefix", 0) // page
    wanted = [max(0, -(-n // page) - prefix) for n in length]
    pages = prefix + sum(wanted) + 5
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)  # pages come from a used pool, in no order
    width = prefix + max(wanted) + 1
    # where each sequence's pages begin in `order`, behind the prefix's; entries past a sequence's last page are never used
    first = torch.tensor([prefix + sum(wanted[:s]) for s in range(rows)], device=dev)
    column = torch.arange(width, device=dev)[None] - prefix
    table = order[(first[:, None] + column).clamp(0, pages - 1)]
    table = torch.where(column < 0, order[:width][None], table).contiguous()
    total = sum(new)
    behind = case.get("behind", 0)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16) * scale)

    state = dict(op=case["op"], q_heads=hq, kv_heads=hkv, page=page, total=total, most_new=max(new), longest=max(length),
                 prefix=prefix * page, prefix_pages=order[:prefix].contiguous(), page_table=table,
                 cu_tokens=torch.tensor([sum(new[:s]) for s in range(rows + 1)], dtype=torch.int32, device=dev),
                 lengths=torch.tensor(length, dtype=torch.int32, device=dev),
                 k_pages=normal(pages, hkv, page, HEAD), v_pages=normal(pages, hkv, page, HEAD, scale=0.5))
    if case["op"] == "append":
        dtype = torch.bfloat16 if case["table"] == "bf16" else torch.float32
        inverse = THETA ** (-torch.arange(0, HEAD, 2, device=dev, dtype=torch.float64) / HEAD)
        angle = (torch.arange(max(length), device=dev, dtype=torch.float64)[:, None] * inverse).repeat(1, 2)
        state.update(qkv=normal(total + behind, (hq + 2 * hkv) * HEAD), q_norm=1 + normal(HEAD, scale=0.1),
                     k_norm=1 + normal(HEAD, scale=0.1), cos=angle.cos().to(dtype), sin=angle.sin().to(dtype),
                     q_out=torch.zeros(total + behind, hq, HEAD, dtype=torch.bfloat16, device=dev))
    else:
        # normalised, rotated queries: a query is nearer to some keys than to most
        state.update(q=normal(total + behind, hq, HEAD, scale=1.5),
                     out=torch.zeros(total + behind, hq * HEAD, dtype=torch.bfloat16, device=dev))
    return state


# ------------------------------------------------------------------------------------- one pass

_framework = None


def _ops():
    global _framework
    if _framework is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "inference-performance-engineering_b200"))
        from ipe_b200 import ops

        _framework = ops
    return _framework


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "decode": _decode, "prefill": _prefill, "shared": _shared}[state["op"]](state)


def _run_own(s):
    ops = _ops()
    if s["op"] == "append":
        ops.paged_qk_norm_rope_append(s["qkv"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], s["cu_tokens"], s["lengths"],
                                      s["page_table"], EPS, s["q_out"], s["k_pages"], s["v_pages"])
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["op"] == "decode":
        return ops.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["out"])
    if s["op"] == "prefill":
        return ops.paged_prefill_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["cu_tokens"], s["lengths"],
                                           s["out"])
    return ops.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix_pages"], s["page_table"], s["lengths"],
                                       s["out"])


def _token_places(s):
    """(sequence, place among the sequence's new tokens, position) of every new token."""
    cu = s["cu_tokens"].long()
    token = torch.arange(s["total"], device=cu.device)
    seq = (cu[1:, None] <= token).sum(0)
    place = token - cu[seq]
    return seq, place, s["lengths"].long()[seq] - (cu[seq + 1] - cu[seq]) + place


def _append(s):
    seq, _, pos = _token_places(s)
    hq, hkv, n = s["q_heads"], s["kv_heads"], s["total"]
    x = s["qkv"][:n].view(n, hq + 2 * hkv, HEAD)
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]

    def rotated(y, weight):
        y = y.float()
        y = weight.float() * (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS))
        return (y * cos + torch.cat((-y[..., HEAD // 2:], y[..., :HEAD // 2]), -1) * sin).to(torch.bfloat16)

    s["q_out"][:n] = rotated(x[:, :hq], s["q_norm"])
    page, row = s["page_table"].long()[seq, pos // s["page"]], pos % s["page"]
    s["k_pages"][page, :, row] = rotated(x[:, hq:hq + hkv], s["k_norm"])
    s["v_pages"][page, :, row] = x[:, hq + hkv:]
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _keys(pages, table, count):
    """fp32 [..., KV heads, count, 128] of the first `count` positions of a page table [..., pages]."""
    page = pages.shape[2]
    x = pages[table[..., :-(-count // page)].long()].transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, HEAD)[..., :count, :].float()


def _weights(score, allowed):
    """exp(score - the row's largest) over the allowed keys, and its sums (1 where a row has no key)."""
    score = score.masked_fill(~allowed, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    e = (score - top).exp()
    return e, e.sum(-1, keepdim=True).masked_fill(~allowed.any(-1, keepdim=True), 1.0)


def _decode(s):
    rows, hq, hkv, most = len(s["lengths"]), s["q_heads"], s["kv_heads"], s["longest"]
    k, v = _keys(s["k_pages"], s["page_table"], most), _keys(s["v_pages"], s["page_table"], most)
    allowed = (torch.arange(most, device=k.device) < s["lengths"][:, None])[:, None, None]
    v = v * allowed[:, :, 0, :, None]
    e, total = _weights(s["q"].view(rows, hkv, -1, HEAD).float() @ k.transpose(-1, -2) * SCALE, allowed)
    s["out"].copy_((e @ v / total).view(rows, hq * HEAD))
    return s["out"]


def _prefill(s):
    hkv, most, group = s["kv_heads"], s["longest"], s["q_heads"] // s["kv_heads"]
    rows, wide, n = len(s["lengths"]), s["most_new"], s["total"]
    cu = s["cu_tokens"].long()
    seq, place, _ = _token_places(s)
    k, v = _keys(s["k_pages"], s["page_table"], most), _keys(s["v_pages"], s["page_table"], most)
    padded = (cu[:-1, None] + torch.arange(wide, device=cu.device)).clamp(max=n - 1)
    q = s["q"][padded].view(rows, wide, hkv, group, HEAD).permute(0, 2, 3, 1, 4).float()
    position = s["lengths"].long()[:, None] - (cu[1:] - cu[:-1])[:, None] + torch.arange(wide, device=cu.device)
    allowed = (torch.arange(most, device=cu.device) <= position[..., None])[:, None, None]
    v = v * (torch.arange(most, device=cu.device) < s["lengths"][:, None])[:, None, :, None]
    e, total = _weights(q @ k[:, :, None].transpose(-1, -2) * SCALE, allowed)
    o = (e @ v[:, :, None] / total).permute(0, 3, 1, 2, 4).reshape(rows, wide, -1)
    s["out"][:n] = o[seq, place].to(torch.bfloat16)
    return s["out"]


def _shared(s):
    rows, hkv, prefix = len(s["lengths"]), s["kv_heads"], s["prefix"]
    most = s["longest"] - prefix
    q = s["q"].view(rows, hkv, -1, HEAD).float()
    k0, v0 = _keys(s["k_pages"], s["prefix_pages"], prefix), _keys(s["v_pages"], s["prefix_pages"], prefix)
    tail = s["page_table"][:, prefix // s["page"]:]
    k1, v1 = _keys(s["k_pages"], tail, most), _keys(s["v_pages"], tail, most)
    key = torch.arange(s["longest"], device=q.device)
    allowed = (key < s["lengths"][:, None])[:, None, None]
    v1 = v1 * allowed[:, :, 0, prefix:, None]
    score = torch.cat((q @ k0.transpose(-1, -2), q @ k1.transpose(-1, -2)), -1) * SCALE
    e, total = _weights(score, allowed)
    s["out"].copy_(((e[..., :prefix] @ v0 + e[..., prefix:] @ v1) / total).view(rows, -1))
    return s["out"]


# -------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    new, length = _sizes(case)
    start = [sum(new[:i]) for i in range(len(new))]
    if case["op"] == "append":
        return _exact_append(s, new, length, start)
    hq, hkv, page = s["q_heads"], s["kv_heads"], s["page"]
    out = s["out"].double()
    for i, (n, total) in enumerate(zip(new, length)):
        if total == 0:
            continue
        row = s["page_table"][i].clone()
        row[:s["prefix"] // page] = s["prefix_pages"]
        row = row[:-(-total // page)].long()
        q = s["q"][start[i]:start[i] + n].double()
        for h in range(hq):
            k = s["k_pages"][row, h * hkv // hq].reshape(-1, HEAD)[:total].double()
            v = s["v_pages"][row, h * hkv // hq].reshape(-1, HEAD)[:total].double()
            score = q[:, h] @ k.T / math.sqrt(HEAD)
            score += torch.full_like(score, -math.inf).triu(total - n + 1)
            out[start[i]:start[i] + n, h * HEAD:(h + 1) * HEAD] = torch.softmax(score, -1) @ v
    return out


def _exact_append(s, new, length, start):
    hq, hkv, page = s["q_heads"], s["kv_heads"], s["page"]
    q_out, k_pages, v_pages = s["q_out"].double(), s["k_pages"].double(), s["v_pages"].double()
    for i, (n, total) in enumerate(zip(new, length)):
        x = s["qkv"][start[i]:start[i] + n].double().view(n, -1, HEAD).transpose(0, 1)
        position = torch.arange(total - n, total, device=x.device)
        c, d = s["cos"][position].double(), s["sin"][position].double()

        def turn(y, w):
            y = y / (y.pow(2).sum(-1, keepdim=True) / HEAD + EPS).sqrt() * w.double()
            a, b = y.chunk(2, -1)
            (c0, c1), (d0, d1) = c.chunk(2, -1), d.chunk(2, -1)
            return torch.cat((a * c0 - b * d0, b * c1 + a * d1), -1)

        q_out[start[i]:start[i] + n] = turn(x[:hq], s["q_norm"]).transpose(0, 1)
        at = s["page_table"][i].long()[position // page] * page + position % page
        for h in range(hkv):
            where = (at // page, torch.full_like(at, h), at % page)
            k_pages[where] = turn(x[hq + h], s["k_norm"])
            v_pages[where] = x[hq + hkv + h]
    return {"q": q_out, "k_pages": k_pages, "v_pages": v_pages}


# ---------------------------------------------------------------------------------------- work

def work(case):
    hq, hkv = case["q_heads"], case["kv_heads"]
    new, length = _sizes(case)
    tokens = sum(new)
    if case["op"] == "append":
        table = HEAD * (2 if case["table"] == "bf16" else 4) * 2
        positions = set()
        for n, total in zip(new, length):
            positions.update(range(total - n, total))
        return {"bytes": 2 * tokens * (hq + 2 * hkv) * HEAD * 2 + len(positions) * table + tokens * 4,
                "flops": tokens * (hq + hkv) * HEAD * 8}
    key_bytes = hkv * HEAD * 2 * 2
    keys = sum(length)
    if case["op"] == "shared":
        keys -= (case["sequences"] - 1) * case["prefix"]
    pairs = sum(n * total - n * (n - 1) // 2 for n, total in zip(new, length))
    return {"bytes": keys * key_bytes + 2 * tokens * hq * HEAD * 2 + keys // case["page"] * 4, "flops": 4 * HEAD * hq * pairs}
