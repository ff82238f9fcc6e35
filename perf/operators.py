"""Cases of the operators that serve several sequences at once.

Four operators, each with its plain form (elementary torch operations, fp32)
and the call a user makes of it:

  packed   causal attention over whole prompts: the rows of several sequences
           packed one after another, grouped heads, optionally after tokens
           that the sequences already hold
  write    new tokens' keys and values into an 8-bit cache held in blocks of
           tokens, one scale for each block and kv head; read back as values
  decode   one token of each sequence over that cache, optionally with the
           attention weight that each block of tokens collected
  evict    the blocks with the least collected weight leave the cache
"""
import math
import random
import sys

import torch

own = False

DEV = "cuda"

# (heads, kv heads, head size): the layer shapes of workloads.py, and two
# generic ones
HEADS = [(14, 2, 64), (32, 32, 128), (32, 8, 128), (28, 4, 128), (16, 2, 64), (8, 8, 128)]


def listed():
    return [
        # three chat turns of a few words
        dict(name="packed_short", op="packed", seqs=3, shortest=1, longest=40, context=0,
             heads=14, kv_heads=2, head_dim=64, spread=1),
        # a batch of ordinary prompts
        dict(name="packed_prompts", op="packed", seqs=8, shortest=60, longest=900, context=0,
             heads=32, kv_heads=8, head_dim=128, spread=2),
        # follow-up turns: new rows after a conversation that is already cached
        dict(name="packed_context", op="packed", seqs=6, shortest=1, longest=500, context=2500,
             heads=28, kv_heads=4, head_dim=128, spread=3),
        # documents
        dict(name="packed_long", op="packed", seqs=4, shortest=2000, longest=5000, context=0,
             heads=32, kv_heads=8, head_dim=128, spread=4),
        # one user, early in the answer
        dict(name="decode_one_short", op="decode", seqs=1, shortest=511, longest=511, block=32,
             heads=14, kv_heads=2, head_dim=64, mass=False, spread=5),
        # one user, far into a long document
        dict(name="decode_one_long", op="decode", seqs=1, shortest=16383, longest=16383, block=32,
             heads=32, kv_heads=8, head_dim=128, mass=False, spread=6),
        # a busy server; the collected weights are kept for a later eviction
        dict(name="decode_batch", op="decode", seqs=64, shortest=17, longest=4000, block=32,
             heads=32, kv_heads=8, head_dim=128, mass=True, spread=7),
        # a model without grouped heads, larger blocks
        dict(name="decode_ungrouped", op="decode", seqs=16, shortest=100, longest=2047, block=64,
             heads=32, kv_heads=32, head_dim=128, mass=False, spread=8),
        # one token of each sequence of a decode step
        dict(name="write_step", op="write", seqs=64, shortest=1, longest=1, filled=4000, block=32,
             kv_heads=8, head_dim=128, spread=9),
        # whole prompts, some after tokens that end inside a block
        dict(name="write_prompts", op="write", seqs=8, shortest=300, longest=4100, filled=100,
             block=32, kv_heads=8, head_dim=128, spread=10),
        # one conversation that has outgrown its share
        dict(name="evict_one", op="evict", seqs=1, shortest=90, longest=90, block=32, keep=64,
             sink=1, recent=4, spread=11),
        # every sequence of a busy server
        dict(name="evict_batch", op="evict", seqs=64, shortest=300, longest=2000, block=32,
             keep=256, sink=2, recent=8, spread=12),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads, head_dim = rng.choice(HEADS)
    spread = rng.randrange(1 << 30)
    op = rng.choice(["packed", "packed", "decode", "decode", "write", "evict"])
    if op == "packed":
        longest, context = log(1, 2500), rng.choice([0, 0, log(1, 2500)])
        most = 25_000_000 // (longest * (longest + 2 * context) // 2 + 1)
        return dict(op=op, seqs=log(1, max(1, min(12, most))), shortest=rng.randint(1, longest),
                    longest=longest, context=context, heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, spread=spread)
    if op == "decode":
        longest = log(1, 12000)
        most = 900_000 // (longest * kv_heads)
        return dict(op=op, seqs=log(1, max(1, min(96, most))),
                    shortest=rng.randint(1, longest), longest=longest, block=rng.choice([32, 32, 64, 128]), heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, mass=rng.random() < 0.5, spread=spread)
    if op == "write":
        longest = log(1, 3000)
        most = 130_000 // (longest * kv_heads)
        return dict(op=op, seqs=log(1, max(1, min(96, most))),
                    shortest=rng.randint(1, longest), longest=longest, filled=log(1, 2000),
                    block=rng.choice([32, 32, 64, 128]), kv_heads=kv_heads, head_dim=head_dim,
                    spread=spread)
    longest = log(8, 1500)
    keep = rng.randint(4, max(4, longest))
    return dict(op=op, seqs=log(1, min(64, 70_000 // longest)),
                shortest=rng.randint(1, longest), longest=longest, block=rng.choice([32, 64, 128]), keep=keep, sink=rng.randint(0, 1),
                recent=rng.randint(1, 3), spread=spread)


# --- sizes of a case: the same for every seed ------------------------------------------------

def _lengths(case, key=0, lo=None, hi=None):
    r = random.Random(case["spread"] * 7 + key)
    lo = case["shortest"] if lo is None else lo
    hi = case["longest"] if hi is None else hi
    n = [r.randint(lo, hi) for _ in range(case["seqs"])]
    if key == 0:
        n[r.randrange(len(n))] = hi
    return n


def _earlier(case):
    """Tokens that each sequence held before the rows of this call."""
    most = case["context"] if case["op"] == "packed" else case["filled"]
    return _lengths(case, 1, 0, most) if most else [0] * case["seqs"]


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# --- inputs ----------------------------------------------------------------------------------

def _pool(g, blocks, kv_heads, block, head_dim):
    """Blocks as a run leaves them: codes of roughly normal values, the largest
    near 127, and scales that differ between blocks and heads."""
    def codes(*shape):
        x = torch.randn(*shape, generator=g, device=DEV)
        return (x * 36.0).clamp_(-127.0, 127.0).round_().to(torch.int8)

    def scales():
        return torch.exp(torch.randn(blocks, kv_heads, generator=g, device=DEV) * 0.3) * 0.028

    return [codes(blocks, kv_heads, block, head_dim), codes(blocks, kv_heads, head_dim, block),
            scales(), scales()]


def _table(g, needed):
    """Each sequence's blocks, in no order, -1 behind its last; and the pool's size."""
    cols, total = max(max(needed), 1), sum(needed)
    pool = total + 3
    ids = torch.randperm(pool, generator=g, device=DEV)[:total].to(torch.int32)
    at = torch.arange(cols, device=DEV)[None, :]
    need = _i32(needed)[:, None]
    first = _i32(_offsets(needed)[:-1])[:, None]
    return torch.where(at < need, ids[(first + at).clamp(max=max(total - 1, 0)).long()],
                       -1).to(torch.int32).contiguous(), pool


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(case)
    if case["op"] == "packed":
        lens, before = _lengths(case), _earlier(case)
        s["q_offsets"] = _i32(_offsets(lens))
        s["k_offsets"] = _i32(_offsets([a + b for a, b in zip(lens, before)]))
        s["longest_q"], s["longest_k"] = max(lens), max(a + b for a, b in zip(lens, before))
        rows, keys = sum(lens), sum(lens) + sum(before)
        # a few dimensions of real queries and keys are larger than the rest
        wide = torch.exp(randn(case["kv_heads"], case["head_dim"]) * 0.3)
        group = case["heads"] // case["kv_heads"]
        s["q"] = randn(rows, case["heads"], case["head_dim"]) * wide.repeat_interleave(group, 0)
        s["k"] = randn(keys, case["kv_heads"], case["head_dim"]) * wide
        s["v"] = randn(keys, case["kv_heads"], case["head_dim"])
    elif case["op"] == "decode":
        lens, block = _lengths(case), case["block"]
        s["table"], pool = _table(g, [-(-n // block) for n in lens])
        s["cache"] = _pool(g, pool, case["kv_heads"], block, case["head_dim"])
        s["lengths"] = _i32(lens)
        s["q"] = randn(case["seqs"], case["heads"], case["head_dim"]) * 1.5
        s["mass_in"] = randn(*s["table"].shape).square() if case["mass"] else None
    elif case["op"] == "write":
        lens, before, block = _lengths(case), _earlier(case), case["block"]
        s["table"], pool = _table(g, [-(-(a + b) // block) for a, b in zip(lens, before)])
        s["cache"] = _pool(g, pool, case["kv_heads"], block, case["head_dim"])
        s["offsets"], s["positions"] = _i32(_offsets(lens)), _i32(before)
        s["k"] = randn(sum(lens), case["kv_heads"], case["head_dim"])
        s["v"] = randn(sum(lens), case["kv_heads"], case["head_dim"])
        # what is read back: the written rows and the earlier ones of their first block
        first = [b // block * block for b in before]
        s["read_positions"] = _i32(first)
        s["read_lens"] = [a + b - f for a, b, f in zip(lens, before, first)]
        s["read_offsets"] = _i32(_offsets(s["read_lens"]))
        s["read_rows"] = sum(s["read_lens"])
        s["touched"] = max(-(-n // block) for n in s["read_lens"])
    else:
        need, block = _lengths(case), case["block"]
        s["table"], _ = _table(g, need)
        r = random.Random(case["spread"] + 5)
        s["lengths"] = _i32([n * block - r.randrange(block) for n in need])
        mass = torch.exp(randn(*s["table"].shape))
        # blocks that no query looked at yet collected nothing
        s["mass"] = torch.where(randn(*mass.shape) > 1.5, 0.0, mass).contiguous()
    return s


# --- the plain forms -------------------------------------------------------------------------

def _padded(offsets, longest):
    """Row of a packed tensor for (sequence, place), and which places are taken."""
    lens = (offsets[1:] - offsets[:-1]).long()
    at = torch.arange(longest, device=DEV)
    taken = at[None, :] < lens[:, None]
    return torch.where(taken, offsets[:-1].long()[:, None] + at[None, :], 0), taken, lens


def _softmax(x, seen):
    """exp(x - max) / sum over the last axis where `seen`, zeros elsewhere."""
    x = torch.where(seen, x, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return torch.where(seen, e / e.sum(-1, keepdim=True), 0.0)


def _plain_packed(s):
    group = s["heads"] // s["kv_heads"]
    qi, q_taken, q_lens = _padded(s["q_offsets"], s["longest_q"])
    ki, _, k_lens = _padded(s["k_offsets"], s["longest_k"])
    n, lq, lk = qi.shape[0], qi.shape[1], ki.shape[1]
    q = s["q"][qi].view(n, lq, s["kv_heads"], group, -1).permute(0, 2, 3, 1, 4)
    k = s["k"][ki].permute(0, 2, 3, 1).unsqueeze(2)
    v = s["v"][ki].permute(0, 2, 1, 3).unsqueeze(2)
    scores = torch.matmul(q * (1.0 / math.sqrt(s["head_dim"])), k)
    last = (k_lens - q_lens)[:, None] + torch.arange(lq, device=DEV)[None, :]
    seen = torch.arange(lk, device=DEV)[None, None, :] <= last[:, :, None]
    w = _softmax(scores, seen[:, None, None])
    out = torch.matmul(w, v).permute(0, 3, 1, 2, 4).reshape(n, lq, s["heads"], -1)
    return out[q_taken]


def _plain_decode(s):
    k_codes, v_codes, k_scales, v_scales = s["cache"]
    ids = s["table"].clamp(min=0).long()
    n, cols = ids.shape
    group, dim, block = s["heads"] // s["kv_heads"], s["head_dim"], s["block"]
    k = k_codes[ids].float() * k_scales[ids][..., None, None]      # n, cols, kv, block, dim
    v = v_codes[ids].float() * v_scales[ids][..., None, None]      # n, cols, kv, dim, block
    k = k.permute(0, 2, 4, 1, 3).reshape(n, s["kv_heads"], dim, cols * block)
    v = v.permute(0, 2, 1, 4, 3).reshape(n, s["kv_heads"], cols * block, dim)
    q = s["q"].view(n, s["kv_heads"], group, dim) * (1.0 / math.sqrt(dim))
    at = torch.arange(cols * block, device=DEV)
    w = _softmax(torch.matmul(q, k), (at[None, :] < s["lengths"][:, None])[:, None, None, :])
    out = torch.matmul(w, v).reshape(n, s["heads"], dim)
    if s["mass_in"] is None:
        return out
    return out, s["mass_in"] + w.sum((1, 2)).view(n, cols, block).sum(-1)


def _plain_requantise(codes, scales, ids, used, new, is_new, is_old):
    """Blocks [n, touched, kv, block, dim]: the scale grows to cover the new rows, the
    earlier codes follow it, rows that hold nothing are 0. Writes the pool; the values.
    Quotients in 64 bits: in 32 some of them round to the other side of a half."""
    old_scale = torch.where(is_old.any(-1)[..., None], scales[ids], 0.0)
    top = torch.where(is_new[:, :, None, :, None], new.abs(), 0.0).amax((-1, -2))
    scale = torch.maximum(old_scale, (top.double() / 127.0).float())
    by = scale[..., None, None]
    moved = codes[ids].double() * old_scale[..., None, None]
    rows = torch.where(is_new[:, :, None, :, None], new.double(),
                       torch.where(is_old[:, :, None, :, None], moved, 0.0))
    fresh = torch.where(by > 0, rows / by, 0.0).round().clamp(-127.0, 127.0).float()
    codes[ids[used]] = fresh[used].to(torch.int8)
    scales[ids[used]] = scale[used]
    return fresh * by


def _plain_write(s):
    k_codes, v_codes, k_scales, v_scales = s["cache"]
    block, touched = s["block"], s["touched"]
    n = s["offsets"].shape[0] - 1
    first = (s["positions"] // block).long()
    lens = (s["offsets"][1:] - s["offsets"][:-1]).long()
    cols = first[:, None] + torch.arange(touched, device=DEV)[None, :]
    used = cols * block < (s["positions"] + lens)[:, None]
    ids = torch.gather(s["table"], 1, cols.clamp(max=s["table"].shape[1] - 1)).clamp(min=0).long()
    place = cols[:, :, None] * block + torch.arange(block, device=DEV)    # n, touched, block
    row = place - s["positions"].long()[:, None, None]
    is_new = (row >= 0) & (row < lens[:, None, None])
    is_old = row < 0
    src = torch.where(is_new, s["offsets"][:-1].long()[:, None, None] + row, 0)
    shape = (n, touched, block, s["kv_heads"], s["head_dim"])
    k_new = s["k"][src.view(-1)].view(shape).transpose(2, 3)
    v_new = s["v"][src.view(-1)].view(shape).transpose(2, 3)
    k = _plain_requantise(k_codes, k_scales, ids, used, k_new, is_new, is_old)
    v = _plain_requantise(v_codes.transpose(2, 3), v_scales, ids, used, v_new, is_new, is_old)
    held = is_new | is_old

    def packed(x):
        return x.transpose(2, 3)[held]

    return packed(k), packed(v)


def _plain_evict(s):
    cols, block = s["table"].shape[1], s["block"]
    blocks = ((s["lengths"] + block - 1) // block).long()[:, None]
    at = torch.arange(cols, device=DEV)[None, :]
    held = at < blocks
    gone = (blocks - s["keep"]).clamp(min=0)
    open_ = held & (at >= s["sink"]) & (at < blocks - s["recent"])
    order = torch.where(open_, s["mass"], math.inf).sort(stable=True, dim=-1).indices
    rank = torch.empty_like(order).scatter_(1, order, at.expand_as(order).contiguous())
    leaves = open_ & (rank < gone)
    stays = held & ~leaves

    def first(mask, values, fill):
        by = (~mask).to(torch.int32).sort(stable=True, dim=-1).indices
        return torch.where(at < mask.sum(-1, keepdim=True), values.gather(1, by), fill)

    return (first(stays, s["table"], -1).to(torch.int32),
            (s["lengths"] - leaves.sum(-1) * block).to(torch.int32),
            first(stays, s["mass"], 0.0), first(leaves, s["table"], -1).to(torch.int32))


def _own(s):
    if "mini-lla_b200" not in sys.path:
        sys.path.insert(0, "mini-lla_b200")
    import mlb

    if s["op"] == "packed":
        return mlb.attention_packed(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"])
    if s["op"] == "evict":
        return mlb.kv8_evict(s["table"], s["lengths"], s["mass"], s["block"], s["keep"],
                             sink_blocks=s["sink"], recent_blocks=s["recent"])
    cache = mlb.Kv8Cache(*s["cache"])
    if s["op"] == "decode":
        if s["mass_in"] is None:
            return mlb.attention_kv8(s["q"], cache, s["table"], s["lengths"])
        mass = torch.empty_like(s["mass_in"])
        out = mlb.attention_kv8(s["q"], cache, s["table"], s["lengths"], mass_in=s["mass_in"],
                                mass_out=mass)
        return out, mass
    mlb.kv8_write(cache, s["table"], s["k"], s["v"], s["offsets"], s["positions"])
    return mlb.kv8_read(cache, s["table"], s["read_offsets"], s["read_positions"], s["read_rows"])


def run(state):
    if own:
        return _own(state)
    return {"packed": _plain_packed, "decode": _plain_decode, "write": _plain_write,
            "evict": _plain_evict}[state["op"]](state)


# --- what a pass cannot do without -----------------------------------------------------------

def work(case):
    if case["op"] == "evict":
        cols, n = max(_lengths(case)), case["seqs"]
        return {"bytes": 4 * (n * (5 * cols) + 2 * n), "flops": 0}
    wide = case["kv_heads"] * case["head_dim"]
    lens = _lengths(case)
    if case["op"] == "packed":
        before = _earlier(case)
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(lens, before))
        rows, keys = sum(lens), sum(lens) + sum(before)
        return {"bytes": 4 * (2 * rows * case["heads"] * case["head_dim"] + 2 * keys * wide),
                "flops": 4 * pairs * case["heads"] * case["head_dim"]}
    blocks = [-(-n // case["block"]) for n in lens]
    if case["op"] == "decode":
        return {"bytes": sum(lens) * 2 * wide + sum(blocks) * (8 * case["kv_heads"] + 4)
                + 8 * case["seqs"] * case["heads"] * case["head_dim"]
                + (8 * sum(blocks) if case["mass"] else 0),
                "flops": 4 * sum(lens) * case["heads"] * case["head_dim"]}
    # write: the new rows in; the codes of the touched blocks out (the earlier
    # ones in too), then the same codes in and their values out
    before, block = _earlier(case), case["block"]
    read = sum(a + b % block for a, b in zip(lens, before))
    old = sum(b % block for b in before)
    return {"bytes": 2 * wide * (4 * sum(lens) + old + read + 5 * read), "flops": 0}


# --- the definition, in 64 bits --------------------------------------------------------------

def _exact_packed(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    qo, ko = s["q_offsets"].tolist(), s["k_offsets"].tolist()
    group = s["heads"] // s["kv_heads"]
    for i in range(s["seqs"]):
        rows, keys = qo[i + 1] - qo[i], ko[i + 1] - ko[i]
        future = torch.ones(rows, keys, dtype=torch.bool, device=DEV).triu(keys - rows + 1)
        for h in range(s["heads"]):
            q = s["q"][qo[i]:qo[i + 1], h].double()
            k = s["k"][ko[i]:ko[i + 1], h // group].double()
            v = s["v"][ko[i]:ko[i + 1], h // group].double()
            x = (q @ k.T / math.sqrt(s["head_dim"])).masked_fill_(future, -math.inf)
            x = x.sub_(x.amax(1, keepdim=True)).exp_()
            out[qo[i]:qo[i + 1], h] = (x @ v) / x.sum(1, keepdim=True)
    return out


def _exact_decode(s):
    k_codes, v_codes, k_scales, v_scales = s["cache"]
    block, kv = s["block"], s["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    mass = s["mass_in"].double() if s["mass_in"] is not None else None
    for i, n in enumerate(s["lengths"].tolist()):
        blocks = -(-n // block)
        ids = s["table"][i, :blocks].long()
        k = torch.cat([k_codes[b].double() * k_scales[b].double()[:, None, None] for b in ids], 1)
        v = torch.cat([v_codes[b].double() * v_scales[b].double()[:, None, None] for b in ids], 2)
        q = s["q"][i].double().view(kv, -1, s["head_dim"])
        x = torch.einsum("hgd,htd->hgt", q, k[:, :n]) / math.sqrt(s["head_dim"])
        x = (x - x.amax(-1, keepdim=True)).exp()
        x = x / x.sum(-1, keepdim=True)
        out[i] = torch.einsum("hgt,hdt->hgd", x, v[:, :, :n]).reshape(s["heads"], -1)
        if mass is not None:
            each = torch.zeros(blocks * block, dtype=torch.float64, device=DEV)
            each[:n] = x.sum((0, 1))
            mass[i, :blocks] += each.view(blocks, block).sum(1)
    return out if mass is None else (out, mass)


def _exact_write(s):
    """Block by block; a scale is what fp32 holds of the largest magnitude / 127."""
    block, table = s["block"], s["table"].tolist()
    offsets, positions = s["offsets"].tolist(), s["positions"].tolist()
    got = []
    for codes, scales, x in ((s["cache"][0], s["cache"][2], s["k"]),
                             (s["cache"][1].transpose(2, 3), s["cache"][3], s["v"])):
        out = []
        for i in range(s["seqs"]):
            at, end = positions[i], positions[i] + offsets[i + 1] - offsets[i]
            for c in range(at // block, -(-end // block)):
                b = table[i][c]
                old = max(0, at - c * block)
                lo, hi = max(at, c * block), min(end, (c + 1) * block)
                new = x[offsets[i] + lo - at:offsets[i] + hi - at].double().transpose(0, 1)
                scale = (new.abs().amax((1, 2)) / 127.0).float().double()
                had = scales[b].double()
                if old:
                    scale = torch.maximum(scale, had)
                rows = torch.cat([codes[b][:, :old].double() * had[:, None, None], new], 1)
                by = scale[:, None, None]
                out.append(((rows / by).round().clamp(-127, 127) * by).transpose(0, 1))
        got.append(torch.cat(out, 0))
    return tuple(got)


def _exact_evict(s):
    """mass_out: the surviving blocks' masses; the rest are whole numbers."""
    mass, lengths = s["mass"].double().cpu(), s["lengths"].tolist()
    out = torch.zeros_like(mass)
    for i, n in enumerate(lengths):
        blocks = -(-n // s["block"])
        open_ = sorted(range(s["sink"], blocks - s["recent"]), key=lambda c: (float(mass[i, c]), c))
        leaves = set(open_[:max(0, blocks - s["keep"])])
        stays = [c for c in range(blocks) if c not in leaves]
        out[i, :len(stays)] = mass[i, stays]
    return (None, None, out, None)


def exact(case, seed):
    s = prepare(case, seed)
    return {"packed": _exact_packed, "decode": _exact_decode, "write": _exact_write,
            "evict": _exact_evict}[s["op"]](s)
