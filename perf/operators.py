"""What is measured of the block operators: routing queries to blocks of a key/value cache, attention over the probed blocks and its
gradients, and eviction from the cache by accumulated attention weight.

A cache row belongs to a block of `block` consecutive rows.  A query row probes `nprobe` blocks, chosen once for the heads that share a
key/value head.  Tensors are [batch][row][head][dim]; a paged cache is [page][row in block][head][dim] with a table block -> page.  Query row t
of a sequence stands at position kv_len - q_len + t and sees the rows up to its own.

`run` computes the operators with elementary torch operations where `own` is false, and with the library's entry points where it is true.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FIRST, LAST = 1, 2          # blocks every query probes: the first of the sequence, and its own with the one before it


# ---------------------------------------------------------------------------------------------------------------------------- cases
def _case(kind, name=None, **kw):
    case = dict(kind=kind, batch=1, q_rows=1, kv_rows=4096, q_heads=32, kv_heads=8, dim=128, block=64, nprobe=16, dtype="bf16", paged=False,
                ragged=False, keep=0)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one sequence answering token by token: latency counts
        _case("route", "route_token", kv_rows=4096),
        # a serving batch of ragged sequences, one token each, blocks are the pages of the cache
        _case("route", "route_batch", batch=64, kv_rows=32768, nprobe=32, paged=True, ragged=True),
        # a whole prompt
        _case("route", "route_prompt", q_rows=8192, kv_rows=8192),
        _case("attend", "attend_token", kv_rows=4096),
        _case("attend", "attend_batch", batch=64, kv_rows=32768, nprobe=32, paged=True, ragged=True),
        _case("attend", "attend_prompt", q_rows=8192, kv_rows=8192),
        # a prompt's next piece on longer caches: odd lengths, three query heads to a key/value head, small blocks
        _case("attend", "attend_piece", batch=3, q_rows=777, kv_rows=5001, q_heads=12, kv_heads=4, dim=96, block=32, nprobe=24, dtype="fp16", ragged=True),
        # a training step's forward and backward pass: a long row of tokens, and a small odd batch with a head of its own for every query head
        _case("train", "train_long", q_rows=8192, kv_rows=8192),
        _case("train", "train_small", batch=2, q_rows=1001, kv_rows=1001, q_heads=8, kv_heads=8, dim=64, block=32, nprobe=8, dtype="fp16"),
        # a serving step adds its attention weights to those of the cache's rows
        _case("weigh", "weigh_batch", batch=64, kv_rows=32768, nprobe=32, paged=True, ragged=True),
        # the cache is cut down: the last queries of a prompt weigh its rows, the heaviest stay
        _case("evict", "evict_short", q_rows=16, kv_rows=2000, keep=1024),
        _case("evict", "evict_long", batch=8, q_rows=128, kv_rows=32768, nprobe=32, keep=8192, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["route", "attend", "train", "weigh", "evict"])
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        kv_heads = rng.choice([1, 2, 4, 8])
        case = _case(kind, q_heads=group * kv_heads, kv_heads=kv_heads, dim=rng.choice([64, 96, 128, 128, 192, 256]), block=rng.choice([16, 32, 64, 64, 128]),
                     nprobe=rng.randint(4, 48), dtype=rng.choice(["bf16", "fp16"]), ragged=rng.random() < 0.5)
        token = kind in ("route", "attend", "weigh") and rng.random() < 0.6
        if kind == "train":
            case["batch"] = rng.randint(1, 4)
            case["q_rows"] = case["kv_rows"] = _log_int(rng, 100, 8192)
        elif token:
            case["batch"] = _log_int(rng, 1, 64)
            case["kv_rows"] = _log_int(rng, 100, 32768)
            case["paged"] = rng.random() < 0.6
        else:
            case["batch"] = rng.randint(1, 8)
            case["kv_rows"] = _log_int(rng, 200, 16384)
            case["q_rows"] = min(case["kv_rows"], _log_int(rng, 2, 128 if kind in ("weigh", "evict") else 8192))
            if kind == "evict":
                case["keep"] = max(64, int(case["kv_rows"] * rng.uniform(0.1, 0.9)))
        logits = case["q_rows"] * case["kv_rows"] * group            # the plain form's largest intermediate, in elements
        rows = case["batch"] * case["kv_rows"] * kv_heads * case["dim"]
        if _cost(case) <= limit and logits <= 3e8 and rows <= 2.2e9:
            return case


# --------------------------------------------------------------------------------------------------------------------------- shapes
def _kv_lens(case):
    """lengths of the sequences in the cache: all the same, or spread from kv_rows down to about half"""
    n, b = case["kv_rows"], case["batch"]
    if not case["ragged"] or b == 1:
        return [n] * b
    return [max(1, n - (i * (n // 2)) // (b - 1)) for i in range(b)]


def _q_lens(case):
    n, b = case["q_rows"], case["batch"]
    lens = _kv_lens(case)
    if not case["ragged"] or b == 1 or n == 1:
        return [min(n, s) for s in lens]
    return [min(s, max(1, n - (i * (n // 4)) // (b - 1))) for i, s in enumerate(lens)]


def _blocks(case):
    return -(-case["kv_rows"] // case["block"])


def _kept(case):
    """rows at the front and at the back of a sequence that an eviction always keeps"""
    return min(4, case["keep"]), min(32, case["keep"] // 2)


def work(case):
    """One pass: each input read once, each output written once; the products of the rows that are probed."""
    B, Hq, Hkv, D, bs, P = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], case["block"], case["nprobe"]
    lens, qlens, kind = _kv_lens(case), _q_lens(case), case["kind"]
    pairs = touched = blocks_seen = 0               # (query row, cache row) pairs; cache rows and block summaries that are needed
    for n, m in zip(lens, qlens):
        union = 0
        for p in range(n - m, n):
            nb = p // bs + 1
            take = min(P, nb)
            pairs += take * bs - (nb * bs - (p + 1))
            blocks_seen += nb
            union += take
        touched += min(n, union * bs)
    q_rows, kv = sum(qlens), sum(lens)
    q_bytes, kv_bytes = q_rows * Hq * D * 2, touched * Hkv * D * 2
    probes = q_rows * Hkv * P * 4
    if kind == "route":
        seen = sum(-(-n // bs) for n in lens)
        fresh = sum(min(n, -(-m // bs) * bs) for n, m in zip(lens, qlens))      # rows of the blocks whose summaries are new
        return {"bytes": q_bytes + fresh * Hkv * D * 2 + seen * Hkv * D * 4 + probes, "flops": 2 * blocks_seen * Hkv * D + q_rows * Hq * D + fresh * Hkv * D}
    if kind == "attend":
        return {"bytes": 2 * q_bytes + 2 * kv_bytes + probes + q_rows * Hq * 4, "flops": 4 * pairs * Hq * D}
    if kind == "train":     # q, k, v, dout in; out, dq, dk, dv out; two products forward, five backward
        return {"bytes": 4 * q_bytes + 4 * kv * Hkv * D * 2 + probes + q_rows * Hq * 4, "flops": 14 * pairs * Hq * D}
    weigh = {"bytes": q_bytes + kv_bytes + probes + q_rows * Hq * 4 + 2 * B * case["kv_rows"] * Hkv * 4, "flops": 2 * pairs * Hq * D}
    if kind == "weigh":
        return weigh
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": weigh["bytes"] + kept * Hkv * (4 * D * 2 + 8), "flops": weigh["flops"]}


# --------------------------------------------------------------------------------------------------------------------------- inputs
def _rows(gen, n, heads, dim, topics, segment, strength):
    """[n][heads][dim]: rows of a text that changes its topic now and then and comes back to earlier ones"""
    x = torch.randn(n, heads, dim, device="cuda", generator=gen)
    return x.add_(topics[:, segment].transpose(0, 1), alpha=strength)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    B, T, Tk, Hq, Hkv, D, bs = (case[x] for x in ("batch", "q_rows", "kv_rows", "q_heads", "kv_heads", "dim", "block"))
    dt, nb = DTYPES[case["dtype"]], _blocks(case)
    lens, qlens = _kv_lens(case), _q_lens(case)
    s = dict(case=case)
    s["q"] = torch.zeros(B, T, Hq, D, device="cuda", dtype=dt)
    if case["paged"]:
        used = [-(-n // bs) for n in lens]
        order = torch.randperm(sum(used), device="cuda", generator=gen).to(torch.int32)
        s["table"] = torch.full((B, nb), -1, device="cuda", dtype=torch.int32)
        s["k"], s["v"] = (torch.zeros(sum(used), bs, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
        at = 0
    else:
        s["table"] = None
        s["k"], s["v"] = (torch.zeros(B, Tk, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
    for b in range(B):
        n, m = lens[b], qlens[b]
        topics = torch.randn(Hkv, 24, D, device="cuda", generator=gen)
        turn = (torch.rand(n, device="cuda", generator=gen) < 1 / 160).cumsum(0)
        segment = torch.randint(24, (n + 1,), device="cuda", generator=gen)[turn]
        k = _rows(gen, n, Hkv, D, topics, segment, 0.5).to(dt)
        v = _rows(gen, n, Hkv, D, topics, segment, 0.25).to(dt)
        s["q"][b, :m] = _rows(gen, m, Hq, D, topics.repeat_interleave(Hq // Hkv, 0), segment[n - m:], 0.6).to(dt)
        if case["paged"]:
            pages = order[at:at + used[b]]
            s["table"][b, :used[b]] = pages
            at += used[b]
            for name, x in (("k", k), ("v", v)):
                full = torch.zeros(used[b] * bs, Hkv, D, device="cuda", dtype=dt)
                full[:n] = x
                s[name][pages.long()] = full.view(used[b], bs, Hkv, D)
        else:
            s["k"][b, :n], s["v"][b, :n] = k, v
    s["kv_len"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
    s["q_len"] = torch.tensor(qlens, device="cuda", dtype=torch.int32)
    if case["kind"] == "train":
        s["dout"] = torch.randn(B, T, Hq, D, device="cuda", generator=gen).to(dt)
        for b in range(B):
            s["dout"][b, qlens[b]:] = 0
    if case["kind"] in ("weigh", "evict"):
        s["mass"] = torch.rand(B, Hkv, Tk, device="cuda", generator=gen) ** 4
    return s


def prepare(case, seed):
    s = _state(case, seed)
    if own:
        _own_prepare(s)
    return s


def _state(case, seed):
    s = _inputs(case, seed)
    kind, B, T, Tk, Hq, Hkv, D, nb, P = case["kind"], *(case[x] for x in ("batch", "q_rows", "kv_rows", "q_heads", "kv_heads", "dim")), _blocks(case), case["nprobe"]
    empty = lambda like: torch.zeros_like(like)
    s["summary"] = torch.zeros(B, Hkv, nb, D, device="cuda")
    s["probes"] = torch.full((B, T, Hkv, P), -1, device="cuda", dtype=torch.int32)
    _plain_summarize(s, s["summary"])                       # a serving program has the summaries of the blocks from its earlier steps
    if kind == "route":
        for b, (n, m) in enumerate(zip(_kv_lens(case), _q_lens(case))):
            s["summary"][b, :, (n - m) // case["block"]:] = 0         # all but those that hold new rows
    else:
        _plain_route(s, s["probes"])
        s["out"], s["lse"] = empty(s["q"]), torch.zeros(B, T, Hq, device="cuda")
    if kind in ("weigh", "evict"):
        s["lse"] = _plain_attend(s)[1]
        s["mass_out"] = empty(s["mass"])
    if kind == "train":
        s["dq"], s["dk"], s["dv"] = empty(s["q"]), empty(s["k"]), empty(s["v"])
    if kind == "evict":
        keep = case["keep"]
        s["kept"], s["count"] = torch.full((B, Hkv, keep), -1, device="cuda", dtype=torch.int32), torch.zeros(B, Hkv, device="cuda", dtype=torch.int32)
        s["k_out"], s["v_out"] = (torch.zeros(B, keep, Hkv, D, device="cuda", dtype=s["k"].dtype) for _ in range(2))
        s["kept_mass"] = torch.zeros(B, Hkv, keep, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------------------------ plain form
def _cache(s, b, name):
    """[rows][heads][dim] of one sequence, in its own type"""
    if s["table"] is None:
        return s[name][b]
    pages = s["table"][b]
    return s[name][pages.clamp(min=0).long()].flatten(0, 1)


def _plain_summarize(s, out, new_rows=None):
    case = s["case"]
    bs = case["block"]
    for b, n in enumerate(_kv_lens(case)):
        lo = 0 if new_rows is None else max(0, n - new_rows[b]) // bs
        hi = -(-n // bs)
        x = _cache(s, b, "k")[lo * bs:n].double()
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, (hi - lo) * bs - x.shape[0])).view(hi - lo, bs, *x.shape[1:]).sum(1)
        rows = (n - torch.arange(lo, hi, device="cuda") * bs).clamp(max=bs).double()
        out[b, :, lo:hi] = (x / rows[:, None, None]).float().transpose(0, 1)
    return out


def _plain_route(s, out):
    case = s["case"]
    bs, P, Hkv = case["block"], case["nprobe"], case["kv_heads"]
    for b, (n, m) in enumerate(zip(_kv_lens(case), _q_lens(case))):
        nb = -(-n // bs)
        q = s["q"][b, :m].double().unflatten(1, (Hkv, -1)).sum(2)                                   # [m][kv head][dim]
        score = torch.matmul(q.transpose(0, 1), s["summary"][b, :, :nb].double().transpose(1, 2))   # [kv head][m][block]
        seen = (torch.arange(n - m, n, device="cuda") // bs + 1)[:, None]
        j = torch.arange(nb, device="cuda")
        score = score.masked_fill((j < FIRST) | (j >= seen - LAST), math.inf).masked_fill(j >= seen, -math.inf)
        order = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :P]
        order = order.masked_fill(order >= seen, nb).sort(-1)[0]                                    # in the order of the cache
        probes = torch.where(order < nb, order, -1)
        out[b, :m, :, :probes.shape[-1]] = probes.transpose(0, 1).to(torch.int32)
    return out


def _tiles(s, lse=None):
    """(sequence, kv head, query rows, cache rows, scale * logits [group][rows][keys] with -inf where a row does not look)"""
    case = s["case"]
    bs, P, Hkv, G = case["block"], case["nprobe"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    for b, (n, m) in enumerate(zip(_kv_lens(case), _q_lens(case))):
        nb = -(-n // bs)
        pos = torch.arange(n - m, n, device="cuda")
        for h in range(Hkv):
            probes = s["probes"][b, :m, h].long()
            heads = slice(h * G, (h + 1) * G)
            k, v = (_cache(s, b, x)[:n, h] for x in ("k", "v"))
            q = s["q"][b, :m, heads].float().transpose(0, 1)
            mask = torch.zeros(m, nb + 1, device="cuda", dtype=torch.bool).scatter_(1, torch.where(probes < 0, nb, probes), True)[:, :nb]
            if m == 1:      # one row: only the rows of its blocks
                keys = (mask[0].nonzero() * bs + torch.arange(bs, device="cuda")).flatten()
                keys = keys[keys < n]
                k, v, seen = k[keys], v[keys], None
            else:
                keys = torch.arange(n, device="cuda")
                seen = mask.repeat_interleave(bs, 1)[:, :n] & (keys <= pos[:, None])
            logits = torch.matmul(q, k.float().t()).mul_(scale)
            yield b, h, m, heads, keys, q, k, v, seen, logits if seen is None else logits.masked_fill_(~seen, -math.inf)


def _plain_attend(s):
    out, lse = torch.zeros_like(s["q"]), torch.zeros_like(s["q"][..., 0], dtype=torch.float32)
    if s["case"]["q_rows"] == 1 and s["case"]["batch"] > 1:
        return _plain_attend_tokens(s, out, lse)
    for b, h, m, heads, keys, q, k, v, seen, logits in _tiles(s):
        top = logits.amax(-1, keepdim=True)
        p = logits.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        out[b, :m, heads] = (torch.matmul(p, v.float()) / total).transpose(0, 1).to(out.dtype)
        lse[b, :m, heads] = (top + total.log())[..., 0].t()
    return out, lse


def _gather_tokens(s, name):
    """one row a sequence: the rows of its probed blocks, [batch][kv head][probe x row in block][dim], and which of them it sees"""
    case = s["case"]
    bs, Hkv = case["block"], case["kv_heads"]
    probes = s["probes"][:, 0].long()                                                              # [batch][kv head][probe]
    rows = (probes.clamp(min=0)[..., None] * bs + torch.arange(bs, device="cuda")).flatten(2)
    seen = (rows < s["kv_len"].long()[:, None, None]) & (probes >= 0).repeat_interleave(bs, 2)
    rows = rows.clamp(max=case["kv_rows"] - 1)
    b, h = torch.arange(rows.shape[0], device="cuda")[:, None, None], torch.arange(Hkv, device="cuda")[None, :, None]
    if s["table"] is None:
        return s[name][b, rows, h], rows, seen
    return s[name][s["table"][b, rows // bs].clamp(min=0).long(), rows % bs, h], rows, seen


def _token_logits(s):
    k, rows, seen = _gather_tokens(s, "k")
    q = s["q"][:, 0].float().unflatten(1, (s["case"]["kv_heads"], -1))
    logits = torch.matmul(q, k.float().transpose(2, 3)).mul_(s["case"]["dim"] ** -0.5)
    return logits.masked_fill_(~seen[:, :, None], -math.inf), rows, seen


def _plain_attend_tokens(s, out, lse):
    logits, rows, seen = _token_logits(s)
    top = logits.amax(-1, keepdim=True)
    p = (logits - top).exp_()
    total = p.sum(-1, keepdim=True)
    v = _gather_tokens(s, "v")[0]
    out[:, 0] = (torch.matmul(p, v.float()) / total).flatten(1, 2).to(out.dtype)
    lse[:, 0] = (top + total.log())[..., 0].flatten(1, 2)
    return out, lse


def _plain_train(s):
    out, lse = torch.zeros_like(s["q"]), torch.zeros_like(s["lse"])
    dq, dk, dv = torch.zeros_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
    scale = s["case"]["dim"] ** -0.5
    for b, h, m, heads, keys, q, k, v, seen, logits in _tiles(s):
        kf, vf = k.float(), v.float()
        top = logits.amax(-1, keepdim=True)
        p = logits.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(total)
        o = torch.matmul(p, vf)
        out[b, :m, heads] = o.transpose(0, 1).to(out.dtype)
        lse[b, :m, heads] = (top + total.log())[..., 0].t()
        do = s["dout"][b, :m, heads].float().transpose(0, 1)
        dv[b, keys, h] = torch.matmul(p.flatten(0, 1).t(), do.flatten(0, 1)).to(dv.dtype)
        ds = torch.matmul(do, vf.t()).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dq[b, :m, heads] = torch.matmul(ds, kf).transpose(0, 1).to(dq.dtype)
        dk[b, keys, h] = torch.matmul(ds.flatten(0, 1).t(), q.flatten(0, 1)).to(dk.dtype)
    return out, dq, dk, dv


def _plain_weigh(s):
    mass = s["mass"].clone()
    if s["case"]["q_rows"] == 1 and s["case"]["batch"] > 1:
        logits, rows, seen = _token_logits(s)
        p = (logits - s["lse"][:, 0].unflatten(1, (s["case"]["kv_heads"], -1))[..., None]).exp_().sum(2)
        return mass.scatter_add_(2, rows, p.masked_fill(~seen, 0))
    for b, h, m, heads, keys, q, k, v, seen, logits in _tiles(s):
        mass[b, h, keys] += (logits - s["lse"][b, :m, heads].t()[..., None]).exp_().sum((0, 1))
    return mass


def _plain_evict(s, mass):
    case = s["case"]
    keep, (first, last) = case["keep"], _kept(case)
    kept, count = torch.full_like(s["kept"], -1), torch.zeros_like(s["count"])
    k_out, v_out, kept_mass = torch.zeros_like(s["k_out"]), torch.zeros_like(s["v_out"]), torch.zeros_like(s["kept_mass"])
    h = torch.arange(case["kv_heads"], device="cuda")[:, None]
    for b, n in enumerate(_kv_lens(case)):
        c = min(n, keep)
        j = torch.arange(n, device="cuda")
        order = torch.sort(mass[b, :, :n].masked_fill((j < first) | (j >= n - last), math.inf), dim=-1, descending=True, stable=True)[1]
        rows = order[:, :c].sort(-1)[0]
        kept[b, :, :c], count[b] = rows.to(torch.int32), c
        k_out[b, :c], v_out[b, :c] = (_cache(s, b, x)[rows, h].transpose(0, 1) for x in ("k", "v"))
        kept_mass[b, :, :c] = mass[b].gather(1, rows)
    return kept, count, k_out, v_out, kept_mass


def run(s):
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "route":
        return _plain_summarize(s, s["summary"], _q_lens(s["case"])), _plain_route(s, s["probes"])
    if kind == "attend":
        return _plain_attend(s)
    if kind == "train":
        return _plain_train(s)
    mass = _plain_weigh(s)
    if kind == "weigh":
        return mass
    return (mass, *_plain_evict(s, s["mass"]))      # by the weight of the steps before: which rows stay does not hang on a sum's last bit


# ------------------------------------------------------------------------------------------------------------------- the library's calls
def _blocks_module():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "gp-ann_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from pygpann import blocks
    return blocks


def _own_prepare(s):
    """the layout of the tensors and the workspace: a program makes them once for its buffers"""
    blocks, case = _blocks_module(), s["case"]
    s["blocks"] = blocks
    s["layout"] = blocks.Layout(
        batch=case["batch"], q_rows=case["q_rows"], kv_rows=case["kv_rows"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["dim"],
        block_rows=case["block"], dtype=case["dtype"], causal=True, scale=case["dim"] ** -0.5, device=torch.cuda.current_device(),
        q_len=s["q_len"].data_ptr(), kv_len=s["kv_len"].data_ptr(), page_table=None if s["table"] is None else s["table"].data_ptr(),
        n_pages=0 if s["table"] is None else s["k"].shape[0], q_stride=s["q"].stride()[:3], k_stride=s["k"].stride()[:3], v_stride=s["v"].stride()[:3])
    calls = {"route": ["route"], "attend": ["attend"], "train": ["attend", "backward"], "weigh": ["weigh"], "evict": ["weigh", "evict"]}[case["kind"]]
    need = blocks.workspace_bytes(s["layout"], case["nprobe"], calls)
    s["workspace"] = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)


def _own_run(s):
    case, blocks, layout, kind = s["case"], s["blocks"], s["layout"], s["case"]["kind"]
    ptr = lambda name: s[name].data_ptr()
    P, stream = case["nprobe"], torch.cuda.current_stream().cuda_stream
    ws = dict(workspace=ptr("workspace"), workspace_bytes=s["workspace"].numel(), stream=stream)
    if kind == "route":
        blocks.summarize(layout, ptr("k"), ptr("summary"), new_rows=case["q_rows"], stream=stream)
        blocks.route(layout, ptr("q"), ptr("summary"), P, ptr("probes"), first=FIRST, last=LAST, **ws)
        return s["summary"], s["probes"]
    if kind in ("attend", "train"):
        blocks.attend(layout, ptr("q"), ptr("k"), ptr("v"), ptr("probes"), P, ptr("out"), ptr("lse"), **ws)
    if kind == "attend":
        return s["out"], s["lse"]
    if kind == "train":
        blocks.attend_backward(layout, ptr("q"), ptr("k"), ptr("v"), ptr("probes"), P, ptr("out"), ptr("lse"), ptr("dout"), ptr("dq"), ptr("dk"), ptr("dv"), **ws)
        return s["out"], s["dq"], s["dk"], s["dv"]
    blocks.weigh(layout, ptr("q"), ptr("k"), ptr("probes"), P, ptr("lse"), ptr("mass"), ptr("mass_out"), **ws)
    if kind == "weigh":
        return s["mass_out"]
    first, last = _kept(case)
    blocks.evict(layout, ptr("k"), ptr("v"), ptr("mass"), case["keep"], ptr("kept"), ptr("count"), ptr("k_out"), ptr("v_out"), ptr("kept_mass"),
                 first=first, last=last, **ws)
    return tuple(s[x] for x in ("mass_out", "kept", "count", "k_out", "v_out", "kept_mass"))


# ------------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definition, row by row of the cache a query looks at, in 64 bits."""
    if work(case)["flops"] > 1e12:
        return None
    s = _state(case, seed)
    f8, dev = torch.float64, "cuda"
    B, T, Tk, Hq, Hkv, D, bs, P = (case[x] for x in ("batch", "q_rows", "kv_rows", "q_heads", "kv_heads", "dim", "block", "nprobe"))
    G, lens, qlens, kind, scale = Hq // Hkv, _kv_lens(case), _q_lens(case), case["kind"], 1 / math.sqrt(D)

    def sequence(name, b):
        if s["table"] is None:
            return s[name][b, :lens[b]].to(f8)
        return torch.cat([s[name][p] for p in s["table"][b].tolist() if p >= 0])[:lens[b]].to(f8)

    if kind == "route":
        summary, probes = s["summary"].to(f8), s["probes"].clone()
        for b in range(B):
            k = sequence("k", b)
            for j in range(max(0, lens[b] - qlens[b]) // bs, -(-lens[b] // bs)):
                summary[b, :, j] = k[j * bs:(j + 1) * bs].mean(0)
            q = s["q"][b, :qlens[b]].to(f8).reshape(qlens[b], Hkv, G, D).sum(2)
            table = summary[b].float().to(f8)
            for h in range(Hkv):
                near = q[:, h] @ table[h].T
                at = torch.arange(lens[b] - qlens[b], lens[b], device=dev)[:, None] // bs
                j = torch.arange(near.shape[1], device=dev)[None]
                near[(j < FIRST) | (at - j < LAST)] = math.inf
                near[j.expand_as(near) > at] = -math.inf
                best = near.argsort(dim=1, descending=True, stable=True)[:, :P].to(torch.int32)
                best = torch.where(best > at, 1 << 30, best).sort(dim=1)[0]
                best[best == 1 << 30] = -1
                probes[b, :qlens[b], h, :best.shape[1]] = best
        return summary, probes

    out, lse = torch.zeros(B, T, Hq, D, device=dev, dtype=f8), torch.zeros(B, T, Hq, device=dev, dtype=f8)
    grads = {x: torch.zeros(s[x].shape, device=dev, dtype=f8) for x in ("dq", "dk", "dv") if x in s}
    mass = s["mass"].to(f8) if "mass" in s else None
    step = max(1, int(6e7 // (P * bs * D)))
    for b in range(B):
        n, m = lens[b], qlens[b]
        k, v = sequence("k", b), sequence("v", b)
        for h in range(Hkv):
            for t in range(0, m, step):
                rows = torch.arange(t, min(m, t + step), device=dev)
                probe = s["probes"][b, rows, h].long()
                key = (probe[:, :, None] * bs + torch.arange(bs, device=dev)).reshape(len(rows), -1)
                sees = (probe >= 0).repeat_interleave(bs, 1) & (key <= (n - m + rows)[:, None])
                key = key.clamp(0, n - 1)
                kk, q = k[key, h], s["q"][b, rows, h * G:(h + 1) * G].to(f8)
                x = (q @ kk.transpose(1, 2) * scale).masked_fill(~sees[:, None], -math.inf)
                z = torch.logsumexp(x, -1)
                if kind in ("weigh", "evict"):
                    p = torch.exp(x - s["lse"][b, rows, h * G:(h + 1) * G].to(f8)[..., None])
                    mass[b, h].index_add_(0, key.flatten(), p.sum(1).flatten())
                    continue
                p = torch.exp(x - z[..., None])
                vv = v[key, h]
                o = p @ vv
                out[b, rows, h * G:(h + 1) * G], lse[b, rows, h * G:(h + 1) * G] = o, z
                if kind == "train":
                    do = s["dout"][b, rows, h * G:(h + 1) * G].to(f8)
                    ds = p * (do @ vv.transpose(1, 2) - (do * o).sum(-1, keepdim=True)) * scale
                    grads["dq"][b, rows, h * G:(h + 1) * G] = ds @ kk
                    grads["dk"][b, :, h].index_add_(0, key.flatten(), (ds.transpose(1, 2) @ q).flatten(0, 1))
                    grads["dv"][b, :, h].index_add_(0, key.flatten(), (p.transpose(1, 2) @ do).flatten(0, 1))
    if kind == "attend":
        return out, lse
    if kind == "train":
        return out, grads["dq"], grads["dk"], grads["dv"]
    if kind == "weigh":
        return mass
    keep, (first, last) = case["keep"], _kept(case)
    kept, count = torch.full((B, Hkv, keep), -1, dtype=torch.int32), torch.zeros(B, Hkv, dtype=torch.int32)
    k_out, v_out, kept_mass = s["k_out"].to(f8), s["v_out"].to(f8), s["kept_mass"].to(f8)
    weights = s["mass"].cpu().tolist()
    for b in range(B):
        n = lens[b]
        k, v = sequence("k", b), sequence("v", b)
        for h in range(Hkv):
            forced = set(range(min(n, first))) | set(range(max(0, n - last), n))
            rows = sorted(forced)[:keep] if n > keep else list(range(n))
            if n > keep:
                rest = sorted((j for j in range(n) if j not in forced), key=lambda j: (-weights[b][h][j], j))
                rows = sorted(rows + rest[:keep - len(rows)])
            kept[b, h, :len(rows)], count[b, h] = torch.tensor(rows, dtype=torch.int32), len(rows)
            at = torch.tensor(rows, device=dev)
            k_out[b, :len(rows), h], v_out[b, :len(rows), h], kept_mass[b, h, :len(rows)] = k[at, h], v[at, h], s["mass"][b, h, at].to(f8)
    return mass, kept.to(dev), count.to(dev), k_out, v_out, kept_mass
