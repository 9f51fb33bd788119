"""Performance cases of the prompt and shared-prefix operators: the calls a serving program makes of them.

``kind`` names the operator:

  prefill  functional.mla_prefill        causal attention of several new tokens per sequence over latent caches
  expand   functional.expand_prefix      a prefix's latent rows into per-head keys and values, kept for its life
  shared   functional.mla_decode_shared  one token per sequence, all of them behind one long prefix

Head dimensions are those of bench.py (latent 512, nope 128, rope 64, value 128); ``heads`` is 128, or fewer where
one GPU holds a share of them. Latents, queries and keys are normal with standard deviation 1, weights
1/sqrt(512). Queries of a prompt come as slices of one projection's output, not yet rotated, in the type that the
model runs in; those of a decode step in float32 and rotated, as functional.mla_decode takes them.
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
MOST_SCORES = 1 << 30  # scores that the plain form and the exact one hold at once


def listed():
    return [
        # a short question to a small share of the heads: three launches' latency is all there is
        {"name": "prompt_f16_1x17_h16", "kind": "prefill", "heads": 16, "dtype": "f16", "batch": 1, "min_new": 17,
         "max_new": 17, "min_old": 0, "max_old": 0, "lens_seed": 0, "block": 0, "prefix": False},
        # one user's page of text, an odd length
        {"name": "prompt_bf16_1x1001", "kind": "prefill", "heads": 128, "dtype": "bf16", "batch": 1, "min_new": 1001,
         "max_new": 1001, "min_old": 0, "max_old": 0, "lens_seed": 0, "block": 0, "prefix": False},
        # a packed batch of documents, each with an opening part that is read in both directions
        {"name": "prompt_bf16_pack12", "kind": "prefill", "heads": 128, "dtype": "bf16", "batch": 12, "min_new": 30,
         "max_new": 2000, "min_old": 0, "max_old": 0, "lens_seed": 3, "block": 0, "prefix": True},
        # one long prompt (the largest)
        {"name": "prompt_bf16_1x8192", "kind": "prefill", "heads": 128, "dtype": "bf16", "batch": 1, "min_new": 8192,
         "max_new": 8192, "min_old": 0, "max_old": 0, "lens_seed": 0, "block": 0, "prefix": False},
        # a piece of each of four prompts, over what 8-bit paged caches hold already; one of eight GPUs that share the heads
        {"name": "chunk_fp8_4x256_h16", "kind": "prefill", "heads": 16, "dtype": "fp8", "batch": 4, "min_new": 256,
         "max_new": 256, "min_old": 1000, "max_old": 8000, "lens_seed": 1, "block": 64, "prefix": False},
        # four drafted tokens of every sequence are checked at once
        {"name": "verify_bf16_16x4", "kind": "prefill", "heads": 128, "dtype": "bf16", "batch": 16, "min_new": 4,
         "max_new": 4, "min_old": 500, "max_old": 6000, "lens_seed": 2, "block": 64, "prefix": False},
        # a system prompt is expanded when the server starts
        {"name": "expand_bf16_1001", "kind": "expand", "heads": 128, "dtype": "bf16", "rows": 1001},
        # a long document of an 8-bit cache, a share of the heads
        {"name": "expand_fp8_8192_h16", "kind": "expand", "heads": 16, "dtype": "fp8", "rows": 8192},
        # two users behind a short prompt
        {"name": "shared_f16_2x512_h16", "kind": "shared", "heads": 16, "dtype": "f16", "batch": 2, "prefix_rows": 512,
         "min_own": 1, "max_own": 60, "lens_seed": 4, "block": 32},
        # a full batch behind a long system prompt
        {"name": "shared_bf16_64x8192", "kind": "shared", "heads": 128, "dtype": "bf16", "batch": 64,
         "prefix_rows": 8192, "min_own": 1, "max_own": 1000, "lens_seed": 5, "block": 64},
        # a few samples of an answer about a long document
        {"name": "shared_bf16_12x32768", "kind": "shared", "heads": 128, "dtype": "bf16", "batch": 12,
         "prefix_rows": 32768, "min_own": 10, "max_own": 300, "lens_seed": 6, "block": 64},
        # many users of one of eight GPUs that share the heads, 8-bit rows, an odd prefix
        {"name": "shared_fp8_200x4001_h16", "kind": "shared", "heads": 16, "dtype": "fp8", "batch": 200,
         "prefix_rows": 4001, "min_own": 0, "max_own": 700, "lens_seed": 7, "block": 64},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["prompt", "chunk", "verify", "expand", "shared"], [4, 2, 2, 2, 4])[0]
    heads, dtype = rng.choice([16, 32, 64, 128, 128]), rng.choice(["bf16", "bf16", "f16", "fp8"])
    lens_seed = rng.randrange(1 << 20)
    if kind == "prompt":
        top = _log_int(rng, 16, 7000)
        batch = _log_int(rng, 1, max(1, min(24, 13000 // top)))
        return {"kind": "prefill", "heads": heads, "dtype": dtype, "batch": batch,
                "min_new": max(1, top // rng.choice([1, 2, 20])), "max_new": top, "min_old": 0, "max_old": 0,
                "lens_seed": lens_seed, "block": rng.choice([0, 0, 64]), "prefix": rng.random() < 0.3}
    if kind == "chunk":
        old = _log_int(rng, 100, 12000)
        batch = _log_int(rng, 1, max(1, min(8, 16000 // old)))
        new = _log_int(rng, 32, 600)
        return {"kind": "prefill", "heads": heads, "dtype": dtype, "batch": batch, "min_new": max(1, new // 2),
                "max_new": new, "min_old": old // 3, "max_old": old, "lens_seed": lens_seed,
                "block": rng.choice([0, 32, 64, 128]), "prefix": False}
    if kind == "verify":
        new, old = rng.randint(1, 8), _log_int(rng, 100, 8000)
        return {"kind": "prefill", "heads": heads, "dtype": dtype, "batch": _log_int(rng, 1, 32), "min_new": new,
                "max_new": new, "min_old": old // 4, "max_old": old, "lens_seed": lens_seed,
                "block": rng.choice([32, 64, 64, 128]), "prefix": False}
    if kind == "expand":
        return {"kind": "expand", "heads": heads, "dtype": dtype, "rows": _log_int(rng, 16, 12000)}
    rows = _log_int(rng, 64, 32768)
    own_rows = _log_int(rng, 1, 1000)
    return {"kind": "shared", "heads": heads, "dtype": dtype, "batch": _log_int(rng, 1, max(1, min(256, 500000 // rows))),
            "prefix_rows": rows, "min_own": own_rows // 8, "max_own": own_rows, "lens_seed": lens_seed,
            "block": rng.choice([32, 64, 64, 128])}


def _lens(case):
    """Of every sequence: (new tokens, rows before them, rows of the opening that is read both ways), from the case alone."""
    r = random.Random(case["lens_seed"])
    if case["kind"] == "shared":
        return [(1, r.randint(case["min_own"], case["max_own"]), 0) for _ in range(case["batch"])]
    lens = [(r.randint(case["min_new"], case["max_new"]), r.randint(case["min_old"], case["max_old"])) for _ in
            range(case["batch"])]
    return [(n, o, r.randint(0, n + o) if case["prefix"] else 0) for n, o in lens]


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


def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads, kind = case["heads"], case["kind"]
    model = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    s = {"case": case, "model": model}
    s["W_UK"] = _randn(g, heads * DN, DC, dtype=model, scale=DC ** -0.5)
    s["W_UV"] = _randn(g, heads * DV, DC, dtype=model, scale=DC ** -0.5)
    if kind == "expand":
        s["rows"] = _randn(g, case["rows"], ROW, dtype=DTYPE[case["dtype"]])
        s["cos"], s["sin"] = _tables(case["rows"])
    else:
        s["lens"] = lens = _lens(case)
        rows = [o + (n if kind == "prefill" else 0) for n, o, _ in lens]
        if case["block"]:
            # a pool with a few blocks more than the sequences hold, in any order; entries past a sequence's rows
            # name block 0
            used = [-(-r // case["block"]) for r in rows]
            order = torch.randperm(sum(used) + 3, generator=g, device="cuda").int().cpu()
            table = torch.zeros(len(rows), max(max(used), 1), dtype=torch.int32)
            at = _cumulative(used)
            for b, n in enumerate(used):
                table[b, :n] = order[at[b]:at[b] + n]
            s["kv"] = _randn(g, order.numel() * case["block"], ROW, dtype=DTYPE[case["dtype"]])
            s["table"] = table.cuda()
            s["seq_lens"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        else:
            s["kv"] = _randn(g, sum(rows), ROW, dtype=DTYPE[case["dtype"]])
            s["seq_offsets"] = torch.tensor(_cumulative(rows), dtype=torch.int32, device="cuda")
            s["row_at"] = _cumulative(rows)
        s["row_count"] = rows
        tokens = sum(n for n, _, _ in lens)
        if kind == "prefill":
            s["q"] = _randn(g, tokens, heads, DN + DR, dtype=model)
            s["token_at"] = _cumulative([n for n, _, _ in lens])
            s["q_offsets"] = torch.tensor(s["token_at"], dtype=torch.int32, device="cuda")
            if case["prefix"]:
                s["both_ways"] = torch.tensor([p for _, _, p in lens], dtype=torch.int32, device="cuda")
            s["cos"], s["sin"] = _tables(max(rows))
        else:
            s["q_nope"] = torch.randn(tokens, heads, DN, generator=g, device="cuda")
            s["q_rope"] = torch.randn(tokens, heads, DR, generator=g, device="cuda")
            s["rows"] = _randn(g, case["prefix_rows"], ROW, dtype=DTYPE[case["dtype"]])
            s["cos"], s["sin"] = _tables(case["prefix_rows"] + max(rows))
    if own:
        latent_attn, F = _functional()
        s["cfg"] = latent_attn.MLAConfig(5120, DC, DN, DR, heads, DV)
        if kind == "shared":
            # made once for a prefix, which thousands of steps read; listed as an operator of its own
            s["prefix"] = F.expand_prefix(s["rows"], s["W_UK"], s["W_UV"], s["cos"], s["sin"], s["cfg"])
    return s


def _run_own(s):
    _, F = _functional()
    kind = s["case"]["kind"]
    if kind == "expand":
        p = F.expand_prefix(s["rows"], s["W_UK"], s["W_UV"], s["cos"], s["sin"], s["cfg"])
        return p.k_nope, p.v, p.k_rope
    cache = {"seq_offsets": s.get("seq_offsets"), "seq_lens": s.get("seq_lens"), "block_table": s.get("table"),
             "block_size": s["case"]["block"]}
    if kind == "prefill":
        return F.mla_prefill(s["kv"], s["q"][..., :DN], s["q"][..., DN:], s["W_UK"], s["W_UV"], s["cos"], s["sin"],
                             s["cfg"], q_offsets=s["q_offsets"], prefix_lens=s.get("both_ways"), rotate_q=True, **cache)
    return F.mla_decode_shared(s["prefix"], s["kv"], s["q_nope"], s["q_rope"], s["W_UK"], s["W_UV"], s["cos"], s["sin"],
                               s["cfg"], out_dtype=s["model"], **cache)


# --- the plain form: decompress, rotate, softmax, weighted sum, in 32 bits ---------------------------------------


def _rotate(x, cos, sin):
    """Pairs (i, i + 32) of the last dimension turned by their row's angles."""
    a, b = x[..., :DR // 2], x[..., DR // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _paged(s, blocks):
    """The pool's rows of these blocks (indexed as bytes, which every type has)."""
    kv = s["kv"]
    pool = kv.view(torch.uint8).view(-1, s["case"]["block"] * ROW * kv.element_size())
    return pool[blocks.long()].view(kv.dtype).reshape(*blocks.shape[:-1], -1, ROW)


def _rows_of(s, b):
    """Sequence b's cache rows, in its order."""
    if "table" in s:
        n = s["row_count"][b]
        return _paged(s, s["table"][b, :-(-n // s["case"]["block"])])[:n]
    return s["kv"][s["row_at"][b]:s["row_at"][b + 1]]


def _tiles(k, v, r):
    """Keys, values and rope keys (rows, .., dims) padded with zeros to tiles of 64 rows, their indices split."""
    pad = -k.shape[0] % 64
    if pad:
        k, v, r = (torch.cat([x, x.new_zeros(pad, *x.shape[1:])]) for x in (k, v, r))
    heads = k.shape[1]
    return (k.reshape(-1, 2, 32, heads, 8, 2, 2, 4), v.reshape(-1, 4, 2, 2, 4, heads, 4, 32),
            r.reshape(-1, 2, 32, 4, 2, 2, 4))


def _decompress(rows, W, heads):
    """c_t W^T per head: (heads, rows, 128)."""
    return torch.matmul(rows[:, :DC], W.float().view(heads, -1, DC).transpose(1, 2))


def _plain_attention(q_nope, q_rope, parts, W_UK, W_UV, limit):
    """q (tokens, heads, .), parts (rows, rotated keys); token t sees the first limit[t] keys (all where None)."""
    heads = q_nope.shape[1]
    rows = torch.cat([r for r, _ in parts])
    k_rope = torch.cat([k for _, k in parts])
    n, keys = q_nope.shape[0], rows.shape[0]
    if keys == 0:
        return q_nope.new_zeros(n, heads, DV)
    out = q_nope.new_empty(n, heads, DV)
    step = max(1, min(heads, MOST_SCORES // (n * keys)))
    seen = None if limit is None else torch.arange(keys, device=rows.device) < limit[:, None]
    for h in range(0, heads, step):
        m = min(step, heads - h)
        K = _decompress(rows, W_UK[h * DN:(h + m) * DN], m)
        V = _decompress(rows, W_UV[h * DV:(h + m) * DV], m)
        score = torch.matmul(q_nope[:, h:h + m].transpose(0, 1), K.transpose(1, 2))
        score += torch.matmul(q_rope[:, h:h + m].transpose(0, 1), k_rope.T)
        score *= SCALE
        if seen is not None:
            score.masked_fill_(~seen, -math.inf)
        score -= score.amax(-1, keepdim=True)
        score.exp_()
        total = score.sum(-1, keepdim=True)
        out[:, h:h + m] = (torch.matmul(score, V) / total).transpose(0, 1)
    return out


def _run_plain(s):
    case = s["case"]
    heads, kind, cos, sin = case["heads"], case["kind"], s["cos"], s["sin"]
    if kind == "expand":
        rows = s["rows"].float()
        return _tiles(_decompress(rows, s["W_UK"], heads).transpose(0, 1).to(s["model"]),
                      _decompress(rows, s["W_UV"], heads).transpose(0, 1).to(s["model"]),
                      _rotate(rows[:, DC:], cos, sin).to(s["model"]))
    outs = []
    if kind == "prefill":
        q = s["q"].float()
        for b, (n, old, both) in enumerate(s["lens"]):
            rows = _rows_of(s, b).float()
            mine = q[s["token_at"][b]:s["token_at"][b + 1]]
            at = torch.arange(old, old + n, device=q.device)
            limit = (at + 1).clamp(min=both)
            q_rope = _rotate(mine[..., DN:], cos[at][:, None], sin[at][:, None])
            k_rope = _rotate(rows[:, DC:], cos[:old + n], sin[:old + n])
            outs.append(_plain_attention(mine[..., :DN], q_rope, [(rows, k_rope)], s["W_UK"], s["W_UV"], limit))
        return torch.cat(outs).to(s["model"])
    # every sequence's keys are the prefix's, decompressed once for all, and its own
    P = case["prefix_rows"]
    front = s["rows"].float()
    front_rope = _rotate(front[:, DC:], cos[:P], sin[:P])
    Kf, Vf = _decompress(front, s["W_UK"], heads), _decompress(front, s["W_UV"], heads)
    score = torch.matmul(s["q_nope"].transpose(0, 1), Kf.transpose(1, 2))
    score += torch.matmul(s["q_rope"].transpose(0, 1), front_rope.T)
    score *= SCALE
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top)
    total, acc = weight.sum(-1, keepdim=True), torch.matmul(weight, Vf)
    q_abs = torch.matmul(s["q_nope"].transpose(0, 1), s["W_UK"].float().view(heads, DN, DC)).transpose(0, 1)
    # the sequences' own rows are few, and padded to the longest: one batch of products in the latent space
    longest = max(s["row_count"])
    if longest == 0:
        return (acc / total).transpose(0, 1).to(s["model"])
    own_rows = _paged(s, s["table"])[:, :longest].float()
    own_rope = _rotate(own_rows[..., DC:], cos[P:P + longest], sin[P:P + longest])
    own_score = torch.matmul(q_abs, own_rows[..., :DC].transpose(1, 2))
    own_score += torch.matmul(s["q_rope"], own_rope.transpose(1, 2))
    own_score *= SCALE
    past = torch.arange(longest, device=score.device) >= s["seq_lens"][:, None]
    own_score.masked_fill_(past[:, None], -math.inf)
    top, total, acc = (x.transpose(0, 1) for x in (top, total, acc))
    both_top = torch.maximum(top, own_score.amax(-1, keepdim=True))
    own_weight = torch.exp(own_score - both_top)
    shrink = torch.exp(top - both_top)
    latent = torch.matmul(own_weight, own_rows[..., :DC])
    mine = torch.matmul(latent.transpose(0, 1), s["W_UV"].float().view(heads, DV, DC).transpose(1, 2)).transpose(0, 1)
    return ((acc * shrink + mine) / (total * shrink + own_weight.sum(-1, keepdim=True))).to(s["model"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --- work and exact values ------------------------------------------------------------------------------------------


def work(case):
    heads = case["heads"]
    size = 1 if case["dtype"] == "fp8" else 2
    weights = heads * (DN + DV) * DC * 2
    if case["kind"] == "expand":
        n = case["rows"]
        return {"bytes": n * ROW * size + weights + n * DR // 2 * 8 + n * (heads * (DN + DV) + DR) * 2,
                "flops": 2 * n * heads * (DN + DV) * DC}
    lens = _lens(case)
    if case["kind"] == "prefill":
        tokens, rows = sum(n for n, _, _ in lens), sum(n + o for n, o, _ in lens)
        # the cheaper of the two forms for every sequence: keys and values decompressed, or queries absorbed
        flops = 0
        for n, o, both in lens:
            seen = sum(max(o + j + 1, both) for j in range(n))
            flops += 2 * heads * min((n + o) * (DN + DV) * DC + seen * (DN + DR + DV),
                                     n * (DN + DV) * DC + seen * (2 * DC + DR))
        return {"bytes": rows * ROW * size + weights + max(n + o for n, o, _ in lens) * DR // 2 * 8 +
                tokens * heads * (DN + DR + DV) * 2, "flops": flops}
    P, batch, own_rows = case["prefix_rows"], case["batch"], sum(o for _, o, _ in lens)
    # the prefix's keys and values are kept decompressed, so its pairs take the fewer products; read as latent rows
    # it is fewer bytes
    return {"bytes": (P + own_rows) * ROW * size + weights + (P + max(o for _, o, _ in lens)) * DR // 2 * 8 +
            batch * heads * ((DN + DR) * 4 + DV * 2),
            "flops": 2 * heads * (batch * P * (DN + DR + DV) + own_rows * (2 * DC + DR) + batch * (DN + DV) * DC)}


def exact(case, seed):
    """The same from the definition in 64 bits, in latent space: scores (q W_UK) c_t + q_rope key, (P c_t) W_UV^T."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    heads, kind = case["heads"], case["kind"]
    cos, sin = s["cos"].double(), s["sin"].double()
    turn = torch.complex(cos, sin)

    def turned(x, at):  # pairs as complex numbers
        z = torch.complex(x[..., :DR // 2].contiguous(), x[..., DR // 2:].contiguous()) * at
        return torch.cat([z.real, z.imag], -1)

    uk, uv = s["W_UK"].double().view(heads, DN, DC), s["W_UV"].double().view(heads, DV, DC)
    if kind == "expand":
        r = s["rows"].double()
        latent = r[:, :DC].T.contiguous()
        k = torch.matmul(s["W_UK"].double(), latent).view(heads, DN, -1).permute(2, 0, 1)
        v = torch.matmul(s["W_UV"].double(), latent).view(heads, DV, -1).permute(2, 0, 1)
        whole = -(-k.shape[0] // 64) * 64  # zeros up to whole tiles, the indices split as SharedPrefix has them
        out = [torch.zeros(whole, *x.shape[1:], dtype=x.dtype, device="cuda") for x in (k, v, r[:, DC:])]
        for x, y in zip(out, (k, v, turned(r[:, DC:], turn))):
            x[:y.shape[0]] = y
        return (out[0].view(-1, 2, 32, heads, 8, 2, 2, 4), out[1].view(-1, 4, 2, 2, 4, heads, 4, 32),
                out[2].view(-1, 2, 32, 4, 2, 2, 4))
    pairs = sum(n * (o + n + case.get("prefix_rows", 0)) for n, o, _ in s["lens"])
    if pairs * heads > 2.0e10:
        return None
    if kind == "prefill":
        q_nope, q_rope = s["q"][..., :DN].double(), s["q"][..., DN:].double()
    else:
        q_nope, q_rope = s["q_nope"].double(), s["q_rope"].double()
    out = torch.zeros(q_nope.shape[0], heads, DV, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, old, both) in enumerate(s["lens"]):
        kv = _rows_of(s, b).double()
        if kind == "shared":
            kv = torch.cat([s["rows"].double(), kv])
        keys = kv.shape[0]
        last = torch.arange(keys - n, keys, device="cuda") if kind == "prefill" else torch.full((n,), keys - 1, device="cuda")
        hidden = torch.arange(keys, device="cuda") > last.clamp(min=both - 1)[:, None]
        k_rope = turned(kv[:, DC:], turn[:keys])
        c = kv[:, :DC].contiguous()
        size = max(1, min(heads, (MOST_SCORES // 4) // max(1, n * keys)))
        for h in range(0, heads, size):
            m = min(size, heads - h)
            qn, qr = q_nope[first:first + n, h:h + m], q_rope[first:first + n, h:h + m]
            if kind == "prefill":
                qr = turned(qr, turn[last][:, None])
            latent_q = torch.matmul(qn.permute(1, 0, 2).contiguous(), uk[h:h + m])  # (m, n, 512)
            x = torch.matmul(latent_q.reshape(m * n, DC), c.T).view(m, n, keys)
            x += torch.matmul(qr.permute(1, 0, 2).reshape(m * n, DR), k_rope.T).view(m, n, keys)
            x = torch.where(hidden, -math.inf, x * SCALE)
            w = torch.exp(x - x.amax(-1, keepdim=True))
            w /= w.sum(-1, keepdim=True)
            lat = torch.matmul(w.view(m * n, keys), c).view(m, n, DC)
            out[first:first + n, h:h + m] = torch.matmul(lat, uv[h:h + m].transpose(1, 2)).permute(1, 0, 2)
        first += n
    return out
