"""Performance cases of the draft-tree and eviction operators: the calls a serving program makes of them.

``kind`` names the operator:

  tree    functional.mla_decode_tree  attention of a tree of drafted tokens per sequence over latent caches
  accept  functional.accept_kv        the accepted path's rows become the sequence's last ones
  weigh   functional.weigh_kv         the attention weight that the newest tokens give every row, summed over steps
  evict   functional.evict_kv         every sequence cut back to its heaviest rows, in place

Head dimensions are those of bench.py (latent 512, nope 128, rope 64, value 128); ``heads`` is 128, or fewer where
one GPU holds a share of them. Latents, queries and keys are normal with standard deviation 1, weights
1/sqrt(512). ``block`` is the block size of a paged cache, or 0 for equal regions. Queries come as slices of one
projection's output in the type that the model runs in, not yet rotated.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
DC, DN, DR, DV = 512, 128, 64, 128
ROW = DC + DR
SCALE = 1.0 / math.sqrt(DN + DR)


def listed():
    return [
        # one user's short draft on a GPU that holds an eighth of the heads: launches' latency
        {"name": "tree_f16_1x7_h16", "kind": "tree", "heads": 16, "dtype": "f16", "batch": 1, "nodes": 7, "min_rows": 500,
         "max_rows": 500, "lens_seed": 0, "block": 0},
        # small trees of a full batch, ragged contexts in a paged cache
        {"name": "tree_bf16_16x16", "kind": "tree", "heads": 128, "dtype": "bf16", "batch": 16, "nodes": 16,
         "min_rows": 500, "max_rows": 6000, "lens_seed": 1, "block": 64},
        # an odd tree over 8-bit rows, a quarter of the heads
        {"name": "tree_fp8_8x25_h32", "kind": "tree", "heads": 32, "dtype": "fp8", "batch": 8, "nodes": 25,
         "min_rows": 1000, "max_rows": 8000, "lens_seed": 2, "block": 32},
        # wide trees over long contexts (the largest)
        {"name": "tree_bf16_4x64", "kind": "tree", "heads": 128, "dtype": "bf16", "batch": 4, "nodes": 64,
         "min_rows": 4000, "max_rows": 16000, "lens_seed": 3, "block": 64},
        # a few tokens accepted in every sequence of a full batch
        {"name": "accept_bf16_64x25", "kind": "accept", "dtype": "bf16", "batch": 64, "nodes": 25, "min_rows": 100,
         "max_rows": 2000, "lens_seed": 4, "block": 64},
        # one user
        {"name": "accept_f16_1x64", "kind": "accept", "dtype": "f16", "batch": 1, "nodes": 64, "min_rows": 1000,
         "max_rows": 1000, "lens_seed": 5, "block": 0},
        # a step of one user
        {"name": "weigh_bf16_1x1001", "kind": "weigh", "heads": 128, "dtype": "bf16", "batch": 1, "tokens": 1,
         "min_rows": 1001, "max_rows": 1001, "lens_seed": 0, "block": 0},
        # a step of the decode benchmark's batch
        {"name": "weigh_bf16_32x8192", "kind": "weigh", "heads": 128, "dtype": "bf16", "batch": 32, "tokens": 1,
         "min_rows": 8192, "max_rows": 8192, "lens_seed": 0, "block": 0},
        # the last tokens of two prompts weigh them before they are cut, a share of the heads
        {"name": "weigh_f16_2x32_h16", "kind": "weigh", "heads": 16, "dtype": "f16", "batch": 2, "tokens": 32,
         "min_rows": 4001, "max_rows": 6000, "lens_seed": 6, "block": 0},
        # many ragged users of 8-bit rows, a share of the heads
        {"name": "weigh_fp8_64x4000_h16", "kind": "weigh", "heads": 16, "dtype": "fp8", "batch": 64, "tokens": 1,
         "min_rows": 300, "max_rows": 4000, "lens_seed": 7, "block": 64},
        # one user's short cache
        {"name": "evict_bf16_1x1001", "kind": "evict", "dtype": "bf16", "batch": 1, "min_rows": 1001, "max_rows": 1001,
         "lens_seed": 0, "block": 0, "keep": 512, "first": 4, "last": 64},
        # the decode benchmark's batch cut to a quarter
        {"name": "evict_bf16_32x8192", "kind": "evict", "dtype": "bf16", "batch": 32, "min_rows": 6000, "max_rows": 8192,
         "lens_seed": 8, "block": 64, "keep": 2048, "first": 4, "last": 256},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["tree", "accept", "weigh", "evict"], [4, 1, 3, 2])[0]
    dtype, block, lens_seed = rng.choice(["bf16", "bf16", "f16"]), rng.choice([0, 32, 64, 128]), rng.randrange(1 << 20)
    if kind == "accept":
        rows = _log_int(rng, 64, 4000)
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, 128), "nodes": rng.randint(2, 64),
                "min_rows": max(64, rows // 4), "max_rows": rows, "lens_seed": lens_seed, "block": block}
    if kind == "evict":
        rows = _log_int(rng, 64, 32768)
        keep = _log_int(rng, max(16, rows // 16), rows)
        first = rng.choice([0, 4, 16])
        return {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, max(1, min(64, 262144 // rows))),
                "min_rows": max(1, rows // rng.choice([1, 2, 8])), "max_rows": rows, "lens_seed": lens_seed,
                "block": block, "keep": keep, "first": first, "last": rng.randint(0, keep - first)}
    heads, dtype = rng.choice([16, 32, 64, 128, 128]), rng.choice(["bf16", "bf16", "f16", "fp8"])
    if kind == "tree":
        nodes = _log_int(rng, 1, 64)
        rows = _log_int(rng, 64, 16000)
        most = min(32, 4 * 64 * 128 * 8000 // (nodes * heads * rows), 128000 // rows)
        return {"kind": kind, "heads": heads, "dtype": dtype, "batch": _log_int(rng, 1, max(1, most)), "nodes": nodes,
                "min_rows": max(64, rows // rng.choice([1, 4])), "max_rows": rows, "lens_seed": lens_seed, "block": block}
    tokens = rng.choice([1, 1, _log_int(rng, 2, 32)])
    rows = _log_int(rng, 64, 32768)
    most = min(64, 32 * 128 * 8192 // (tokens * heads * rows), 262144 // rows)
    return {"kind": kind, "heads": heads, "dtype": dtype, "batch": _log_int(rng, 1, max(1, most)), "tokens": tokens,
            "min_rows": max(64, rows // rng.choice([1, 8])), "max_rows": rows, "lens_seed": lens_seed, "block": block}


def _lens(case):
    """Rows of every sequence, from the case alone (a tree's own rows among them)."""
    r = random.Random(case["lens_seed"])
    return [r.randint(case["min_rows"], case["max_rows"]) for _ in range(case["batch"])]


def _trees(case):
    """Of every sequence its nodes' parents (-1: a child of the last token) and a path from the top, from the case
    alone: nodes attach to one of the few before them, as a drafter's best candidates do."""
    r = random.Random(case["lens_seed"] + 1)
    n = case["nodes"]
    parents = [[-1 if j == 0 else r.randint(max(-1, j - 6), j - 1) for j in range(n)] for _ in range(case["batch"])]
    paths = []
    for p in parents:
        leaf, path = r.randrange(n), []
        while leaf >= 0:
            path.insert(0, leaf)
            leaf = p[leaf]
        paths.append((path + [-1] * n)[:n])
    return parents, paths


def _functional():
    path = os.path.abspath("latent-attn_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import latent_attn
    from latent_attn import functional

    return latent_attn, functional


def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _tables(rows):
    """cos and sin of position * 10000^(-2i/64), float32."""
    freq = 10000.0 ** (-torch.arange(0, DR, 2, dtype=torch.float64, device="cuda") / DR)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, batch = case["kind"], case["batch"]
    model = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    lens = _lens(case)
    s = {"case": case, "model": model, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    s["seq_lens"] = s["lens"].clone()  # (accept and evict change these; the next step of the program fills them again)
    if case["block"]:
        # a pool with a few blocks more than the sequences hold, in any order; entries past a sequence's rows name block 0
        used = [-(-n // case["block"]) for n in lens]
        order = torch.randperm(sum(used) + 3, generator=g, device="cuda").int().cpu()
        table = torch.zeros(batch, -(-case["max_rows"] // case["block"]), dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        s["kv"] = _randn(g, order.numel() * case["block"], ROW, dtype=DTYPE[case["dtype"]])
        s["table"] = table.cuda()
        s["room"] = table.shape[1] * case["block"]
    else:
        s["room"] = case["max_rows"]
        s["kv"] = _randn(g, batch, s["room"], ROW, dtype=DTYPE[case["dtype"]])
    if kind in ("tree", "accept"):
        parents, paths = _trees(case)
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
        s["path"] = torch.tensor(paths, dtype=torch.int32, device="cuda")
    if kind in ("tree", "weigh"):
        tokens = batch * (case["nodes"] if kind == "tree" else case["tokens"])
        s["q"] = _randn(g, tokens, case["heads"], DN + DR, dtype=model)
        s["W_UK"] = _randn(g, case["heads"] * DN, DC, dtype=model, scale=DC ** -0.5)
        s["cos"], s["sin"] = _tables(max(lens))
    if kind == "tree":
        s["W_UV"] = _randn(g, case["heads"] * DV, DC, dtype=model, scale=DC ** -0.5)
    if kind == "weigh":
        s["weights"] = torch.zeros(batch, s["room"], device="cuda")
    if kind == "evict":
        # what some thousand steps leave: most rows get little, a few a lot; some exactly alike
        x = torch.randn(batch, s["room"], generator=g, device="cuda").mul_(2).exp_()
        s["weighed"] = torch.where(x < 0.05, 0.0, x)
        s["weights"] = s["weighed"].clone()
    return s


def _run_own(s):
    latent_attn, F = _functional()
    case, kind = s["case"], s["case"]["kind"]
    cfg = latent_attn.MLAConfig(5120, DC, DN, DR, case.get("heads", 128), DV)
    cache = {"block_table": s.get("table"), "block_size": case["block"]}
    if kind == "tree":
        return F.mla_decode_tree(s["kv"], s["q"][..., :DN], s["q"][..., DN:], s["W_UK"], s["W_UV"], s["cos"], s["sin"], cfg,
                                 s["parents"], seq_lens=s["seq_lens"], rotate_q=True, **cache)
    if kind == "weigh":
        F.weigh_kv(s["weights"], s["kv"], s["q"][..., :DN], s["q"][..., DN:], s["W_UK"], s["cos"], s["sin"], cfg,
                   seq_lens=s["seq_lens"], rotate_q=True, **cache)
        return s["weights"]
    if kind == "accept":
        F.accept_kv(s["kv"], s["seq_lens"], case["nodes"], s["path"], cfg, **cache)
        return s["kv"], s["seq_lens"]
    kept = F.evict_kv(s["kv"], s["seq_lens"], s["weights"], cfg, case["keep"], first=case["first"], last=case["last"], **cache)
    return s["kv"], s["seq_lens"], s["weights"], kept


# --- the plain form: rows gathered, absorbed queries, softmax, weighted sum, in 32 bits ------------------------------


def _rotate(x, cos, sin):
    """Pairs (i, i + 32) of the last dimension turned by their row's angles."""
    a, b = x[..., :DR // 2], x[..., DR // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _places(s):
    """Where every position of every sequence lies in the cache, (batch, room)."""
    at = torch.arange(s["room"], device="cuda")
    if "table" not in s:
        return at + s["room"] * torch.arange(s["case"]["batch"], device="cuda")[:, None]
    block = s["case"]["block"]
    return s["table"].long()[:, at // block] * block + at % block


def _flat(s):
    return s["kv"].view(-1, ROW)


def _rows(s):
    """All sequences' rows, padded to the longest, float32 (batch, room, 576); indexed as bytes, which every type has."""
    size = s["kv"].element_size()
    return _flat(s).view(torch.uint8).view(-1, ROW * size)[_places(s)].view(s["kv"].dtype).float()


def _scores(s, rows, q, q_at, k_at):
    """Base-e scores (batch, tokens * heads, room) of q (batch, tokens, heads, 192) at positions q_at over keys at k_at."""
    heads, cos, sin = s["case"]["heads"], s["cos"], s["sin"]
    batch, n = q.shape[:2]
    nope = q[..., :DN].reshape(batch * n, heads, DN).transpose(0, 1)
    latent = torch.matmul(nope, s["W_UK"].float().view(heads, DN, DC)).transpose(0, 1).reshape(batch, n * heads, DC)
    rope = _rotate(q[..., DN:], cos[q_at][:, :, None], sin[q_at][:, :, None]).reshape(batch, n * heads, DR)
    keys = _rotate(rows[..., DC:], cos[k_at], sin[k_at])
    x = torch.matmul(torch.cat([latent, rope], -1), torch.cat([rows[..., :DC], keys], -1).transpose(1, 2).contiguous())
    return x * SCALE


def _ancestors(parents):
    """(batch, n, n): whether node j is node i or one of its ancestors, and every node's depth."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    step = (parents[..., None] == at) | (at[:, None] == at)
    seen = torch.linalg.matrix_power(step.float(), 64) > 0  # (64 nodes at most; counts stay below infinity)
    return seen, seen.sum(-1) - 1


def _softmax(x, hidden):
    x = x.masked_fill_(hidden, -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    return x


def _plain_tree(s):
    heads, n, batch = s["case"]["heads"], s["case"]["nodes"], s["case"]["batch"]
    rows = _rows(s)
    at = torch.arange(s["room"], device="cuda")
    before = (s["lens"].long() - n)[:, None]
    seen, depth = _ancestors(s["parents"])
    # of every position the node there, and its place in the text: its index, or the context's length and its depth
    node = at - before
    inside = (node >= 0) & (node < n)
    node = node.clamp(0, n - 1)
    k_at = torch.where(inside, before + depth.gather(1, node), at).clamp(max=s["cos"].shape[0] - 1)
    x = _scores(s, rows, s["q"].float().view(batch, n, heads, DN + DR), before + depth, k_at)
    mask = (at < before)[:, None] | (inside[:, None] & seen.gather(2, node[:, None].expand(-1, n, -1)))
    x = _softmax(x.view(batch, n, heads, -1), ~mask[:, :, None]).view(batch, n * heads, -1)
    latent = torch.matmul(x, rows[..., :DC].contiguous()).view(batch * n, heads, DC).transpose(0, 1)
    out = torch.matmul(latent, s["W_UV"].float().view(heads, DV, DC).transpose(1, 2).contiguous())
    return out.transpose(0, 1).to(s["model"])


def _plain_weigh(s):
    heads, n, batch = s["case"]["heads"], s["case"]["tokens"], s["case"]["batch"]
    rows = _rows(s)
    at = torch.arange(s["room"], device="cuda")
    q_at = (s["lens"].long() - n)[:, None] + torch.arange(n, device="cuda")
    x = _scores(s, rows, s["q"].float().view(batch, n, heads, DN + DR), q_at, at.clamp(max=s["cos"].shape[0] - 1))
    x = _softmax(x.view(batch, n, heads, -1), (at > q_at[..., None])[:, :, None])
    s["weights"] += x.sum((1, 2))
    return s["weights"]


def _plain_accept(s):
    n = s["case"]["nodes"]
    kv, places, path = _flat(s), _places(s), s["path"].long()
    size, first = kv.element_size(), (s["lens"].long() - n)[:, None]
    taken = path >= 0
    src = places.gather(1, first + path.clamp(min=0))
    dst = places.gather(1, first + torch.arange(n, device="cuda"))
    kv = kv.view(torch.uint8).view(-1, ROW * size)
    kv[dst[taken]] = kv[src[taken]]
    s["seq_lens"].copy_(s["lens"] - n + taken.sum(1))
    return s["kv"], s["seq_lens"]


def _plain_evict(s):
    case, w = s["case"], s["weights"]
    keep, lens = case["keep"], s["lens"].long()[:, None]
    at = torch.arange(s["room"], device="cuda")
    filled = at < lens
    stays = (at < case["first"]) | (at >= lens - case["last"])
    order = torch.where(filled, torch.where(stays, math.inf, w), -math.inf).sort(dim=1, descending=True, stable=True).indices
    # the filled rows come first: past their number nothing is kept
    most = torch.minimum(lens, torch.full_like(lens, keep))
    rank = torch.arange(s["room"], device="cuda").expand_as(order)
    mask = torch.zeros_like(filled).scatter_(1, order, rank < most)
    kept = torch.where(mask, at, s["room"]).sort(dim=1).values[:, :keep]
    valid = kept < s["room"]
    from_at = kept.clamp(max=s["room"] - 1)
    kv, places = _flat(s), _places(s)
    kv = kv.view(torch.uint8).view(-1, ROW * kv.element_size())
    kv[places[:, :keep][valid]] = kv[places.gather(1, from_at)[valid]]
    moved = w.gather(1, from_at)
    w.masked_fill_(filled, 0.0)
    w[:, :keep] = torch.where(valid, moved, w[:, :keep])
    s["seq_lens"].copy_(most[:, 0])
    return s["kv"], s["seq_lens"], w, torch.where(valid, kept, -1).int()


_PLAIN = {"tree": _plain_tree, "accept": _plain_accept, "weigh": _plain_weigh, "evict": _plain_evict}


def run(state):
    kind = state["case"]["kind"]
    # a cache that was cut is filled again before it is cut the next time: its lengths and weights are
    if kind in ("accept", "evict"):
        state["seq_lens"].copy_(state["lens"])
    if kind == "evict":
        state["weights"].copy_(state["weighed"])
    return _run_own(state) if own else _PLAIN[kind](state)


# --- work and exact values ------------------------------------------------------------------------------------------


def work(case):
    size = 1 if case["dtype"] == "fp8" else 2
    kind, lens = case["kind"], _lens(case)
    if kind == "accept":
        moved = sum(sum(p >= 0 for p in path) for path in _trees(case)[1])
        return {"bytes": moved * ROW * size * 2 + case["batch"] * (4 * case["nodes"] + 8), "flops": 0}
    if kind == "evict":
        # rows that stay where they are need not move: the first ones, and all of a short sequence
        cut = [n for n in lens if n > case["keep"]]
        return {"bytes": len(cut) * (case["keep"] - case["first"]) * (ROW * size * 2 + 4) + sum(lens) * 4 +
                sum(cut) * 4 + case["batch"] * (4 * case["keep"] + 8), "flops": 0}
    heads = case["heads"]
    if kind == "weigh":
        n = case["tokens"]
        pairs = sum(n * r - n * (n - 1) // 2 for r in lens)
        tokens = n * len(lens)
        return {"bytes": sum(lens) * (ROW * size + 8) + heads * DN * DC * 2 + max(lens) * DR * 4 +
                tokens * heads * (DN + DR) * 2, "flops": 2 * heads * (pairs * ROW + tokens * DN * DC)}
    n = case["nodes"]
    depths = 0
    for parents in _trees(case)[0]:
        d = []
        for p in parents:
            d.append(d[p] + 1 if p >= 0 else 1)
        depths += sum(d)
    pairs, tokens = sum(n * (r - n) for r in lens) + depths, n * len(lens)
    return {"bytes": sum(lens) * ROW * size + heads * (DN + DV) * DC * 2 + max(lens) * DR * 4 +
            tokens * heads * (DN + DR + DV) * 2, "flops": 2 * heads * (pairs * (2 * DC + DR) + tokens * (DN + DV) * DC)}


def exact(case, seed):
    """From the definition in 64 bits, a sequence at a time: keys and values decompressed, rows moved one after another."""
    s = prepare(case, seed)
    kind, lens = case["kind"], _lens(case)
    flat = s["kv"].view(-1, ROW)

    def places(b):  # of sequence b's positions
        if case["block"]:
            return torch.cat([torch.arange(case["block"], device="cuda") + case["block"] * int(i) for i in s["table"][b].tolist()])
        return torch.arange(s["room"], device="cuda") + b * s["room"]

    if kind in ("accept", "evict"):
        out, w = flat.clone(), s.get("weights")
        new_lens, kepts = [], []
        for b, L in enumerate(lens):
            at = places(b)
            if kind == "accept":
                take = [L - case["nodes"] + p for p in s["path"][b].tolist() if p >= 0]
                to = L - case["nodes"]
            else:
                x = w[b, :L].tolist()
                take, to = list(range(L)), 0
                if L > case["keep"]:
                    middle = sorted(range(case["first"], L - case["last"]), key=lambda i: (-x[i], i))
                    take = sorted(list(range(case["first"])) + middle[:case["keep"] - case["first"] - case["last"]] +
                                  list(range(L - case["last"], L)))
                w[b, :L] = 0
                w[b, :len(take)] = torch.tensor([x[i] for i in take], device="cuda")
                kepts.append(take + [-1] * (case["keep"] - len(take)))
            out[at[to:to + len(take)]] = flat[at[torch.tensor(take, dtype=torch.long, device="cuda")]]
            new_lens.append(to + len(take))
        n = torch.tensor(new_lens, dtype=torch.int32, device="cuda")
        out = out.view(s["kv"].shape).double()
        return (out, n) if kind == "accept" else (out, n, w.double(), torch.tensor(kepts, dtype=torch.int32, device="cuda"))

    heads = case["heads"]
    n = case["nodes"] if kind == "tree" else case["tokens"]
    cos, sin = s["cos"].double(), s["sin"].double()
    uk = s["W_UK"].double().view(heads, DN, DC)
    uv = s["W_UV"].double().view(heads, DV, DC) if kind == "tree" else None
    size = s["kv"].element_size()
    outs = []
    weights = s["weights"].double() if kind == "weigh" else None

    def turned(x, at):  # pairs as complex numbers
        z = torch.complex(x[..., :DR // 2].contiguous(), x[..., DR // 2:].contiguous()) * torch.complex(cos[at], sin[at])
        return torch.cat([z.real, z.imag], -1)

    for b, L in enumerate(lens):
        kv = flat.view(torch.uint8).view(-1, ROW * size)[places(b)[:L]].view(flat.dtype).double()
        key_at = torch.arange(L, device="cuda")
        sees = torch.zeros(n, L, dtype=torch.bool)
        if kind == "tree":
            q_at = []
            for j, p in enumerate(s["parents"][b].tolist()):
                if p >= 0:
                    sees[j] = sees[p]
                else:
                    sees[j, :L - n] = True
                sees[j, L - n + j] = True
                q_at.append(int(sees[j].sum()) - 1)
            key_at[L - n:] = torch.tensor(q_at, device="cuda")
            q_at = torch.tensor(q_at, device="cuda")
        else:
            for j in range(n):
                sees[j, :L - n + j + 1] = True
            q_at = torch.arange(L - n, L, device="cuda")
        sees = sees.cuda()
        q = s["q"][b * n:(b + 1) * n].double()
        rope = turned(q[..., DN:], q_at[:, None].expand(-1, heads))
        keys = turned(kv[:, DC:], key_at)
        c = kv[:, :DC].contiguous()
        out = torch.empty(n, heads, DV, dtype=torch.float64, device="cuda")
        step = max(1, min(heads, (1 << 27) // (L * max(n, DN))))
        for h in range(0, heads, step):
            m = min(step, heads - h)
            K = torch.matmul(c, uk[h:h + m].reshape(m * DN, DC).T).view(L, m, DN).permute(1, 2, 0).contiguous()
            x = torch.matmul(q[:, h:h + m, :DN].transpose(0, 1).contiguous(), K)
            x += torch.matmul(rope[:, h:h + m].transpose(0, 1).contiguous(), keys.T)
            x = (x * SCALE).masked_fill(~sees, -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            x /= x.sum(-1, keepdim=True)
            if kind == "weigh":
                weights[b, :L] += x.sum((0, 1))
            else:
                V = torch.matmul(c, uv[h:h + m].reshape(m * DV, DC).T).view(L, m, DV).transpose(0, 1).contiguous()
                out[:, h:h + m] = torch.matmul(x, V).transpose(0, 1)
        outs.append(out)
    return weights if kind == "weigh" else torch.cat(outs)
