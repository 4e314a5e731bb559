"""Operators for several continuations of one prompt, measured against their plain forms.

A serving program that keeps n continuations of a prompt (best of n, beams,
drafts to rank) forks cache pages (``copy_blocks``), decodes sequences that
share their first pages (``hip_shared_decode``) and scores the tokens it drew
(``token_logprobs``). Heads and layers are those of ``microinfer_amd.workloads``
and ``microinfer_amd.engine.model`` (8 KV heads of 128, 16 or 32 query heads,
28 layers, blocks of 16, a vocabulary of 151936) or generic odd ones.

Lengths, page lists and their placement come from the case alone (``lens``
seeds them), values from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 16
HEAD_DIM = 128
VOCAB = 151936
LAYERS = 4  # attention layers that run on one step's plan
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One stream's next token with the five best alternatives, as an API answers it.
        dict(name="logprob_decode_1", kind="logprob", dtype="bf16", rows=1, vocab=VOCAB, given=1,
             top=5, heat=False, entropy=False, pad=0),
        # A decode batch at temperatures, twenty alternatives and the entropy of each choice.
        dict(name="logprob_decode_64", kind="logprob", dtype="bf16", rows=64, vocab=VOCAB, given=1,
             top=20, heat=True, entropy=True, pad=0),
        # Scoring a chunk of prompt tokens: no alternatives, the logits of 3000 positions.
        dict(name="logprob_prompt", kind="logprob", dtype="bf16", rows=3000, vocab=VOCAB, given=1,
             top=0, heat=False, entropy=True, pad=0),
        # Float32 logits of an odd vocabulary inside wider rows, eight choices scored in each.
        dict(name="logprob_f32_odd", kind="logprob", dtype="f32", rows=333, vocab=32003, given=8,
             top=8, heat=False, entropy=True, pad=5),
        # Forking one sequence: its partial last page, in every layer.
        dict(name="fork_1", kind="copy", dtype="bf16", layers=28, heads=8, dim=128, block=BLOCK,
             layout="paired", parents=1, pairs=1, whole=False, lens=1),
        # Beam search moving 8 survivors' last pages to 64 beams.
        dict(name="fork_64", kind="copy", dtype="bf16", layers=28, heads=8, dim=128, block=BLOCK,
             layout="paired", parents=8, pairs=64, whole=False, lens=2),
        # Compaction of a fragmented pool: whole pages, every layer. The largest copy.
        dict(name="compact_1000", kind="copy", dtype="bf16", layers=28, heads=8, dim=128,
             block=BLOCK, layout="paired", parents=1000, pairs=1000, whole=True, lens=3),
        # A small float32 pool with tokens outermost and an odd number of heads.
        dict(name="copy_f32_tokens", kind="copy", dtype="f32", layers=5, heads=3, dim=64, block=32,
             layout="token_major", parents=40, pairs=77, whole=False, lens=4),
        # Four drafts of a short prompt: launch latency counts.
        dict(name="shared_4_short", kind="shared", dtype="bf16", hq=16, hkv=8, groups=1, per=4,
             prefix_lo=500, prefix_hi=500, tail_lo=1, tail_hi=60, lens=5),
        # Best of 16 on a long document.
        dict(name="shared_16_long", kind="shared", dtype="bf16", hq=32, hkv=8, groups=1, per=16,
             prefix_lo=12000, prefix_hi=12000, tail_lo=1, tail_hi=500, lens=6),
        # A batch of prompts of different lengths, several drafts of each, in half precision.
        dict(name="shared_groups_f16", kind="shared", dtype="f16", hq=16, hkv=8, groups=6, per=7,
             prefix_lo=300, prefix_hi=3000, tail_lo=5, tail_hi=300, lens=7),
        # 64 requests behind one system prompt. The largest attention.
        dict(name="shared_64_system", kind="shared", dtype="bf16", hq=32, hkv=8, groups=1, per=64,
             prefix_lo=3500, prefix_hi=3500, tail_lo=20, tail_hi=700, lens=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case, at most as much work as the largest listed one of its kind."""
    while True:
        case = _draw(rng)
        most = max(_cost(c) for c in listed() if c["kind"] == case["kind"])
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _draw(rng):
    kind = rng.choice(["logprob", "copy", "shared"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    lens = rng.randrange(1 << 20)
    if kind == "logprob":
        vocab = rng.choice([VOCAB, VOCAB, _log(rng, 40, 260000)])
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 3000), vocab=vocab,
                    given=rng.choice([1, 1, rng.randint(2, 12)]),
                    top=rng.choice([0, 1, 5, 20, rng.randint(1, 32)]), heat=rng.random() < 0.4,
                    entropy=rng.random() < 0.6, pad=rng.choice([0, 0, 0, rng.randint(1, 40)]))
    if kind == "copy":
        whole = rng.random() < 0.4
        pairs = _log(rng, 1, 1000)
        return dict(kind=kind, dtype=dtype, layers=rng.choice([1, 28, rng.randint(1, 36)]),
                    heads=rng.choice([8, 8, 4, rng.randint(1, 12)]),
                    dim=rng.choice([128, 128, 64, 8 * rng.randint(2, 32)]),
                    block=rng.choice([16, 16, 32, 64]),
                    layout=rng.choice(["paired", "paired", "head_major", "token_major"]),
                    parents=pairs if whole else _log(rng, 1, pairs), pairs=pairs, whole=whole,
                    lens=lens)
    groups = rng.randint(1, 8)
    per = _log(rng, 1, 64)
    lo = _log(rng, 16, 12000)
    tail = _log(rng, 1, 300)
    return dict(kind=kind, dtype=dtype if dtype != "f32" or rng.random() < 0.4 else "bf16",
                hq=rng.choice([16, 32, 32, 8, 64]), hkv=8, groups=groups, per=per, prefix_lo=lo,
                prefix_hi=_log(rng, lo, 2 * lo), tail_lo=tail, tail_hi=_log(rng, tail, 3 * tail),
                lens=lens)


# ---------------------------------------------------------------------------
# Lists and lengths (from the case).
# ---------------------------------------------------------------------------
def _page_lists(case):
    """Sources, destinations and leading tokens of a copy, and the pool's pages."""
    rng = random.Random(case["lens"])
    pool = 2 * case["pairs"] + 3
    ids = rng.sample(range(pool), case["parents"] + case["pairs"])
    parents, dst = ids[:case["parents"]], ids[case["parents"]:]
    if case["whole"]:
        return parents, dst, None, pool
    src = [parents[i % case["parents"]] for i in range(case["pairs"])]
    fill = {p: rng.randint(1, case["block"] - 1) for p in parents}
    return src, dst, [fill[s] for s in src], pool


def _lengths(case):
    """Per group the shared tokens (whole pages), per sequence the whole context."""
    rng = random.Random(case["lens"])
    shared, contexts = [], []
    for _ in range(case["groups"]):
        prefix = rng.randint(case["prefix_lo"], case["prefix_hi"])
        shared.append(prefix // BLOCK * BLOCK)
        contexts.append([prefix + rng.randint(case["tail_lo"], case["tail_hi"])
                         for _ in range(case["per"])])
    return shared, contexts


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "logprob":
        rows, vocab, given, top = case["rows"], case["vocab"], case["given"], case["top"]
        out = rows * (4 * given + 12 * top + 4 * case["entropy"])
        return {"bytes": rows * vocab * es + rows * (8 * given + 4 * case["heat"]) + out,
                "flops": rows * vocab * (6 if case["entropy"] else 4)}
    if case["kind"] == "copy":
        src, _, tokens, _ = _page_lists(case)
        row = 2 * case["layers"] * case["heads"] * case["dim"] * es
        tokens = tokens or [case["block"]] * len(src)
        read = sum(dict(zip(src, tokens)).values())
        return {"bytes": row * (read + sum(tokens)), "flops": 0}
    shared, contexts = _lengths(case)
    rows = sum(p + sum(c - p for c in group) for p, group in zip(shared, contexts))
    seqs = case["groups"] * case["per"]
    every = sum(sum(group) for group in contexts)
    hq, hkv = case["hq"], case["hkv"]
    bytes_ = LAYERS * (rows * 2 * hkv * HEAD_DIM * es + 2 * seqs * hq * HEAD_DIM * es)
    return {"bytes": bytes_ + 4 * rows // BLOCK, "flops": LAYERS * 4 * every * hq * HEAD_DIM}


# ---------------------------------------------------------------------------
# Inputs (values from the seed).
# ---------------------------------------------------------------------------
def _pool(layers, blocks, block, heads, dim, layout, dtype, gen):
    """K and V pools as logical [layers, blocks, block, heads, dim] views."""
    if layout == "paired":
        store = torch.randn(layers, blocks, heads, 2, block, dim, generator=gen, device="cuda",
                            dtype=dtype)
        return [store[:, :, :, i].permute(0, 1, 3, 2, 4) for i in (0, 1)]
    if layout == "head_major":
        return [torch.randn(layers, blocks, heads, block, dim, generator=gen, device="cuda",
                            dtype=dtype).permute(0, 1, 3, 2, 4) for _ in (0, 1)]
    return [torch.randn(layers, blocks, block, heads, dim, generator=gen, device="cuda",
                        dtype=dtype) for _ in (0, 1)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["kind"] == "logprob":
        rows, vocab, given = case["rows"], case["vocab"], case["given"]
        logits = torch.randn(rows, vocab + case["pad"], generator=gen, device="cuda")
        logits *= 2.5
        # A few likely tokens in each row, as a trained model's logits have.
        few = torch.randint(vocab, (rows, 12), generator=gen, device="cuda")
        logits.scatter_add_(1, few, 9 * torch.rand(rows, 12, generator=gen, device="cuda"))
        state["logits"] = logits.to(dtype)[:, :vocab]
        tokens = torch.randint(vocab, (rows, given), generator=gen, device="cuda")
        tokens[:, 0] = few[:, 0]
        state["tokens"] = tokens[:, 0].contiguous() if given == 1 else tokens
        state["temperatures"] = None
        if case["heat"]:
            state["temperatures"] = 0.3 + 1.2 * torch.rand(rows, generator=gen, device="cuda")
        return state
    if case["kind"] == "copy":
        src, dst, tokens, blocks = _page_lists(case)
        state["keys"], state["values"] = _pool(case["layers"], blocks, case["block"],
                                               case["heads"], case["dim"], case["layout"], dtype,
                                               gen)
        state.update(src=src, dst=dst, tokens=tokens)
        return state
    shared, contexts = _lengths(case)
    flat = [c for group in contexts for c in group]
    width = max(-(-c // BLOCK) for c in flat)
    rng = random.Random(case["lens"] + 1)
    need = sum(p // BLOCK for p in shared) + sum(-(-c // BLOCK) for c in flat)
    ids = iter(rng.sample(range(need), need))
    tables = []
    for p, group in zip(shared, contexts):
        head = [next(ids) for _ in range(p // BLOCK)]
        for c in group:
            row = head + [next(ids) for _ in range(-(-c // BLOCK) - len(head))]
            tables.append(row + [-1] * (width - len(row)))
    state["keys"], state["values"] = _pool(LAYERS, need, BLOCK, case["hkv"], HEAD_DIM, "paired",
                                           dtype, gen)
    state["query"] = torch.randn(LAYERS, len(flat), case["hq"], HEAD_DIM, generator=gen,
                                 device="cuda", dtype=dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    state.update(tables=ints(tables), contexts=ints(flat),
                 starts=ints([g * case["per"] for g in range(case["groups"] + 1)]),
                 shared=ints([p // BLOCK for p in shared]))
    return state


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def run(state):
    return {"logprob": _run_logprob, "copy": _run_copy, "shared": _run_shared}[
        state["case"]["kind"]](state)


def _run_logprob(state):
    case, logits, tokens = state["case"], state["logits"], state["tokens"]
    if own:
        from microinfer_amd.layer.hip_logprobs import token_logprobs

        got = token_logprobs(logits, tokens, top=case["top"], entropy=case["entropy"],
                             temperatures=state["temperatures"])
        return [x for x in (got.logprobs, got.entropy, got.top_tokens, got.top_logprobs)
                if x is not None]
    x = logits.float()
    if state["temperatures"] is not None:
        x = x / state["temperatures"][:, None]
    x = x - x.amax(1, keepdim=True)
    p = x.exp()
    total = p.sum(1, keepdim=True)
    log_total = total.log()
    given = tokens.view(len(tokens), -1)
    out = [(x.gather(1, given) - log_total).view(tokens.shape)]
    if case["entropy"]:
        out.append((log_total - (p * x).sum(1, keepdim=True) / total)[:, 0])
    if case["top"]:
        # Equal values in the order of their index: the index is part of the key.
        bits = logits.float().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = key * (1 << 32) + torch.arange(logits.shape[1], 0, -1, device=logits.device)
        best = logits.shape[1] - (key.topk(case["top"], 1).values & 0xFFFFFFFF)
        out += [best, x.gather(1, best) - log_total]
    return out


def _run_copy(state):
    keys, values = state["keys"], state["values"]
    if own:
        from microinfer_amd.worker.hip_kv_blocks import copy_blocks

        copy_blocks(keys, values, state["src"], state["dst"], tokens=state["tokens"])
        return [keys, values]
    src = torch.tensor(state["src"], device=keys.device)
    dst = torch.tensor(state["dst"], device=keys.device)
    if state["tokens"] is None:
        keys[:, dst] = keys[:, src]
        values[:, dst] = values[:, src]
        return [keys, values]
    tokens = torch.tensor(state["tokens"], device=keys.device)
    taken = (torch.arange(keys.shape[2], device=keys.device) < tokens[:, None])[..., None, None]
    keys[:, dst] = torch.where(taken, keys[:, src], keys[:, dst])
    values[:, dst] = torch.where(taken, values[:, src], values[:, dst])
    return [keys, values]


def _run_shared(state):
    query, keys, values, tables = (state[k] for k in ("query", "keys", "values", "tables"))
    layers, seqs, hq, dim = query.shape
    hkv = keys.shape[3]
    if own:
        from microinfer_amd.layer.hip_shared_decode import hip_shared_decode, shared_decode_plan

        plan = shared_decode_plan(state["contexts"], state["starts"], state["shared"],
                                  num_q_heads=hq, num_kv_heads=hkv, head_dim=dim,
                                  dtype=query.dtype, block_size=keys.shape[2],
                                  block_table_width=tables.shape[1])
        return [hip_shared_decode(query[i], keys[i], values[i], tables, state["contexts"],
                                  plan=plan) for i in range(layers)]
    pages = tables.clamp(min=0).long()
    # [layers, seqs, pages, block, hkv, dim] -> [layers, seqs, hkv, tokens, dim]
    k = keys[:, pages].permute(0, 1, 4, 2, 3, 5).float().reshape(layers, seqs, hkv, -1, dim)
    q = query.float().view(layers, seqs, hkv, hq // hkv, dim)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(dim)
    del k
    there = torch.arange(scores.shape[-1], device=query.device) < state["contexts"][:, None]
    scores = scores.masked_fill(~there[:, None, None], -math.inf)
    scores = scores - scores.amax(-1, keepdim=True)
    p = scores.exp()
    p = p / p.sum(-1, keepdim=True)
    v = values[:, pages].permute(0, 1, 4, 2, 3, 5).float().reshape(layers, seqs, hkv, -1, dim)
    out = torch.matmul(p, v).view(layers, seqs, hq, dim).to(query.dtype)
    return [out[i] for i in range(layers)]


# ---------------------------------------------------------------------------
# The definitions in 64 bits.
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "logprob":
        return _exact_logprob(case, state)
    if case["kind"] == "copy":
        return _exact_copy(case, state)
    outs = []
    for layer in range(LAYERS):
        rows = []
        for s, c in enumerate(state["contexts"].tolist()):
            at = state["tables"][s, : -(-c // BLOCK)].long()
            k = state["keys"][layer, at].double().flatten(0, 1)[:c]
            v = state["values"][layer, at].double().flatten(0, 1)[:c]
            share = case["hq"] // case["hkv"]
            q = state["query"][layer, s].double().view(case["hkv"], share, HEAD_DIM)
            weights = torch.softmax(q @ k.permute(1, 2, 0).contiguous() * HEAD_DIM ** -0.5, -1)
            rows.append((weights @ v.transpose(0, 1).contiguous()).reshape(case["hq"], HEAD_DIM))
        outs.append(torch.stack(rows))
    return outs


def _exact_logprob(case, state):
    lps, entropies, tops, top_lps = [], [], [], []
    for r0 in range(0, case["rows"], 256):
        raw = state["logits"][r0:r0 + 256].double()
        logp = raw
        if case["heat"]:
            logp = raw / state["temperatures"][r0:r0 + 256, None].double()
        logp = torch.log_softmax(logp, 1)
        tokens = state["tokens"][r0:r0 + 256]
        lps.append(logp.gather(1, tokens.view(len(tokens), -1)).view(tokens.shape))
        if case["entropy"]:
            entropies.append(-(logp.exp() * logp).sum(1))
        if case["top"]:
            order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            tops.append(order)
            top_lps.append(logp.gather(1, order))
    return [torch.cat(x) for x in (lps, entropies, tops, top_lps) if x]


def _exact_copy(case, state):
    keys, values = state["keys"], state["values"]
    tokens = state["tokens"] or [case["block"]] * len(state["src"])
    pairs = list(zip(state["src"], state["dst"], tokens))
    for pool in (keys, values):
        before = {s: pool[:, s].clone() for s in set(state["src"])}
        for s, d, n in pairs:
            pool[:, d, :n] = before[s][:, :n]
    return [keys, values]
