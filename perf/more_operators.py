"""Workloads of the adapters of many requests beside the shared projections (the plan of a step's rows by adapter,
what the adapters add to a projection) and of the log probabilities that a step answers with (of given tokens, with
entropy and top alternatives), each with its plain form in elementary torch operations and its values in 64 bits.

Projections are those of Qwen3-30B-A3B (hidden 2048, 32 query and 4 kv heads of 128) and Qwen3-235B-A22B (4096, 64
and 4), the vocabulary that of both (151936), and a few generic sizes.  An adapter of rank r has, for each part of a
projection (q, k and v are parts of one), A [r, K] and B [columns of the part, r].
"""

from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

own = False  # false: the plain forms; true: the library's operators

HEAD = 128
VOCAB = 151936
RANKS = [8, 16, 32, 64]


def _package():
    """``inference-server_amd/`` of the working folder, imported as ``inference_server_amd``."""
    name = "inference_server_amd"
    if name in sys.modules:
        return sys.modules[name]
    folder = os.path.join(os.getcwd(), "inference-server_amd")
    spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                  submodule_search_locations=[folder])
    mod = importlib.util.module_from_spec(spec)
    sys.modules[name] = mod
    try:
        spec.loader.exec_module(mod)
    except BaseException:
        sys.modules.pop(name, None)
        raise
    return mod


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def _rows(op, seqs, adapters, lo, hi, lens, **more):
    """`seqs` sequences of lo .. hi rows, each with one of `adapters` adapters or (one in eight) none; `lens` seeds
    the lengths and the choice."""
    return {**more, "op": op, "seqs": seqs, "adapters": adapters, "new_lo": lo, "new_hi": hi, "lens": lens}


def _add(seqs, adapters, lo, hi, lens, proj, rank, **more):
    """proj: "qkv" or "o" of a model with `hidden` and `heads` (4 kv heads); rank: the pool's, the adapters' own are
    up to it."""
    return _rows("add", seqs, adapters, lo, hi, lens, proj=proj, rank=rank, **more)


def _logprobs(tokens, vocab, top, dtype="bf16", banned=False, **more):
    return {**more, "op": "logprobs", "tokens": tokens, "vocab": vocab, "top": top, "dtype": dtype, "banned": banned}


SMALL, LARGE = {"hidden": 2048, "heads": 32}, {"hidden": 4096, "heads": 64}


def listed():
    return [
        # a decode step of 64 sequences, most with an adapter of their own: planned once a step
        _rows("plan", 64, 100, 1, 1, 1, name="plan_decode_b64"),
        # a step of prompts of eight tenants: adapters by sequence, rows by the sequences' offsets
        _rows("plan", 12, 8, 100, 1300, 2, name="plan_prompts_b12"),
        # one user's single token behind the output projection, where latency counts
        _add(1, 1, 1, 1, 3, "o", 16, **SMALL, name="add_o_decode_b1"),
        # a decode batch of 24 sequences with adapters of several ranks, beside q, k and v
        _add(24, 16, 1, 1, 4, "qkv", 64, **SMALL, name="add_qkv_decode_b24"),
        # a large decode batch on the large model, nearly every sequence with an adapter of its own
        _add(128, 100, 1, 1, 5, "qkv", 16, **LARGE, name="add_qkv_decode_b128"),
        # prompts of a few tenants in one step
        _add(6, 4, 200, 1500, 6, "qkv", 64, **SMALL, name="add_qkv_prompts_b6"),
        # completions of one policy in training, scored at full batch on the large model
        _add(16, 2, 300, 700, 7, "o", 32, **LARGE, name="add_o_prompts_b16"),
        # one sampled token with its five alternatives, as a chat client asks for
        _logprobs(1, VOCAB, 5, name="logprobs_decode_b1"),
        # a decode batch with twenty alternatives each, some tokens banned
        _logprobs(64, VOCAB, 20, banned=True, name="logprobs_decode_b64"),
        # a prompt scored with alternatives, fp32 logits, a vocabulary that is not a multiple of anything
        _logprobs(777, 50257, 8, dtype="fp32", name="logprobs_prompt_777"),
        # completions scored for preference data: the given tokens and the entropy alone
        _logprobs(6000, VOCAB, 0, name="logprobs_score_6000"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "add", "add", "add", "logprobs", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([VOCAB, _log_int(rng, 1000, 262144)])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        most = 6000 * VOCAB // (vocab * (2 if dtype == "fp32" else 1))
        top = rng.choice([0, 1, 5, 20, rng.randint(1, 64)])
        tokens = _log_int(rng, 1, min(most, 6000 if top == 0 else 1500))
        return _logprobs(tokens, vocab, top, dtype, rng.random() < 0.3)
    decode = rng.random() < 0.5
    seqs = _log_int(rng, 1, 256 if decode else 24)
    adapters = _log_int(rng, 1, 128)
    hi = 1 if decode else _log_int(rng, 1, 8192 // seqs)
    lo = max(1, hi // rng.choice([1, 4, 64]))
    lens = rng.randrange(1 << 30)
    if op == "plan":
        return _rows(op, seqs, adapters, lo, hi, lens)
    shape = rng.choice([SMALL, SMALL, LARGE, {"hidden": 1024, "heads": 12}, {"hidden": 2560, "heads": 20}])
    rank = rng.choice([16, 16, 32, 64, 128])
    return _add(seqs, min(adapters, 32) if rank > 32 else adapters, lo, hi, lens, rng.choice(["qkv", "o"]), rank, **shape)


def _lens(case):
    """(rows, adapter or -1) of each sequence."""
    rng = random.Random(case["lens"])
    return [(rng.randint(case["new_lo"], case["new_hi"]),
             -1 if rng.random() < 0.125 and case["seqs"] > 1 else rng.randrange(case["adapters"]))
            for _ in range(case["seqs"])]


def _projection(case):
    """(K, the parts' columns)"""
    hidden, heads = case["hidden"], case["heads"] * HEAD
    return (hidden, [heads, 4 * HEAD, 4 * HEAD]) if case["proj"] == "qkv" else (heads, [hidden])


def _ranks(case):
    rng = random.Random(case["lens"] + 1)
    return [min(case["rank"], rng.choice(RANKS + [case["rank"]] * 2)) for _ in range(case["adapters"])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    st = {"op": case["op"]}
    if own:
        st["pkg"] = _package()
    if case["op"] == "logprobs":
        return st | _logits(case, seed, gen, dev)

    seqs, L = _lens(case), case["adapters"]
    n, ids = [s[0] for s in seqs], [s[1] for s in seqs]
    # which adapter has which number is another matter each time
    names = torch.randperm(L, generator=torch.Generator().manual_seed(seed)).tolist()
    ids = torch.tensor([names[i] if i >= 0 else -1 for i in ids], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    T = sum(n)
    st |= {"T": T, "L": L, "ids": ids, "cu": cu if max(n) > 1 else None}
    if case["op"] == "plan":
        return st

    K, parts = _projection(case)
    P, R = len(parts), case["rank"]
    rank = torch.tensor(_ranks(case), dtype=torch.int32, device=dev)[torch.tensor(names, device=dev).argsort()]  # by number

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    # a trained adapter's A is of the size that it was drawn with, its B small; alpha is twice the rank
    a, b = normal(L, P, R, K) * K ** -0.5, normal(L, sum(parts), R) * 0.05
    live = torch.arange(R, device=dev) < rank[:, None]
    st["a"] = (a * live[:, None, :, None]).to(torch.bfloat16).view(L, P * R, K)
    st["b"] = (b * live[:, None, :]).to(torch.bfloat16)
    st |= {"rank": rank, "scale": torch.full((L,), 2.0, device=dev), "parts": parts,
           "row_ids": torch.repeat_interleave(ids, torch.tensor(n, device=dev), output_size=T),
           "x": normal(T, K).to(torch.bfloat16), "y": normal(T, sum(parts)).to(torch.bfloat16)}
    if own:  # a program loads its adapters once, and plans a step once for all layers
        st["pool"] = st["pkg"].LoraPool(st["a"], st["b"], st["rank"], st["scale"], tuple(parts))
        st["plan"] = st["pkg"].lora_plan(ids, L, cu_rows=st["cu"], num_rows=T)
    return st


def _logits(case, seed, gen, dev):
    T, V = case["tokens"], case["vocab"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    x = torch.empty((T, V), dtype=dtype, device=dev)
    favourite = torch.randint(0, V, (T,), generator=gen, device=dev)
    sure = torch.rand((T,), generator=gen, device=dev) * 12 + 6  # from undecided rows to sure ones
    some = torch.randint(0, V, (T, 40), generator=gen, device=dev)
    for lo in range(0, T, 512):  # a few hundred rows at a time, in 32 bits
        part = torch.randn((min(512, T - lo), V), generator=gen, device=dev) * 2.2
        part.scatter_add_(1, some[lo:lo + 512], torch.rand((len(part), 40), generator=gen, device=dev) * 9)
        part.scatter_(1, favourite[lo:lo + 512, None], sure[lo:lo + 512, None])
        if case["banned"]:  # tokens that a grammar rules out
            part.masked_fill_(torch.rand((1, V), generator=gen, device=dev) < 0.4, -math.inf)
        x[lo:lo + 512] = part
    # mostly what the model would say, some other tokens, and rows of padding
    kind = torch.rand((T,), generator=gen, device=dev)
    other = torch.randint(0, V, (T,), generator=gen, device=dev)
    tokens = torch.where(kind < 0.7, favourite, other)
    if T > 1:
        tokens = torch.where(kind > 0.95, -1, tokens)
    return {"x": x, "tokens": tokens, "top": case["top"]}


# ---------------------------------------------------------------------------
# the operators, and their plain forms
# ---------------------------------------------------------------------------


def run(st):
    if own:
        return _run_own(st)
    return {"plan": _plain_plan, "add": _plain_add, "logprobs": _plain_logprobs}[st["op"]](st)


def _run_own(st):
    pkg, op = st["pkg"], st["op"]
    if op == "plan":
        plan = pkg.lora_plan(st["ids"], st["L"], cu_rows=st["cu"], num_rows=st["T"])
        return {"rows": plan.rows, "offsets": plan.offsets}
    if op == "add":
        return pkg.lora_add(st["y"], st["x"], st["pool"], st["plan"])
    r = pkg.token_logprobs(st["x"], st["tokens"], st["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    return out | {"top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if st["top"] else out


def _plain_plan(st):
    ids, L, T = st["ids"], st["L"], st["T"]
    if st["cu"] is not None:
        row = torch.arange(T, dtype=torch.int32, device=ids.device)
        ids = ids[torch.searchsorted(st["cu"][1:], row, right=True)]
    key = torch.where((ids >= 0) & (ids < L), ids, L)
    order = torch.sort(key, stable=True).indices.to(torch.int32)
    counts = (key[:, None] == torch.arange(L + 1, device=ids.device)).sum(0)
    return {"rows": order, "offsets": torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)}


def _plain_add(st):
    a, b, y = st["a"].float(), st["b"].float(), st["y"]
    L, PR, K = a.shape
    R = b.shape[2]
    P, T = PR // R, len(y)
    live = torch.arange(R, device=y.device) < st["rank"][:, None]
    mine = st["row_ids"][:, None] == torch.arange(L, device=y.device)
    gain = torch.where(mine[:, :, None] & live, st["scale"][:, None], 0.0)  # [T, L, R]
    u = torch.matmul(st["x"].float(), a.view(L * PR, K).T).view(T, L, P, R) * gain[:, :, None]
    b = b.split(st["parts"], 1)
    delta = [torch.matmul(u[:, :, p].reshape(T, L * R), b[p].transpose(1, 2).reshape(L * R, -1)) for p in range(P)]
    y.copy_(y.float() + torch.cat(delta, 1))
    return y


def _plain_logprobs(st):
    x, tokens, top = st["x"].float(), st["tokens"], st["top"]
    V = x.shape[1]
    shifted = x - x.amax(1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(1)
    entropy = total.log() - (e * torch.where(e > 0, shifted, 0.0)).sum(1) / total
    given = shifted.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0] - total.log()
    out = {"logprobs": torch.where(tokens < 0, 0.0, torch.where(tokens < V, given, math.nan)), "entropy": entropy}
    if not top:
        return out
    # values as whole numbers of the same order, the lower index first among equals
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32
    key = torch.topk(order + (V - 1 - torch.arange(V, device=x.device)), top, dim=1).values
    ids = V - 1 - (key & 0xffffffff)
    return out | {"top_ids": ids, "top_logprobs": shifted.gather(1, ids) - total.log()[:, None]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    if case["op"] == "logprobs":
        T, V, top = case["tokens"], case["vocab"], case["top"]
        size = 2 if case["dtype"] == "bf16" else 4
        # per value: a difference, its exponential, two sums and a product
        return {"bytes": T * (V * size + 8 + 2 * 4 + top * (8 + 4)), "flops": 5 * T * V}
    seqs, L = _lens(case), case["adapters"]
    T = sum(n for n, _ in seqs)
    if case["op"] == "plan":
        return {"bytes": 4 * (T + L + 2 + (2 * len(seqs) + 1 if max(n for n, _ in seqs) > 1 else T)), "flops": 0}
    K, parts = _projection(case)
    N, P, ranks = sum(parts), len(parts), _ranks(case)
    with_adapter = sum(n for n, i in seqs if i >= 0)
    used = sum(ranks[i] for i in {i for _, i in seqs if i >= 0})
    flops = sum(2 * n * ranks[i] * (P * K + N) for n, i in seqs if i >= 0)
    return {"bytes": 4 * T + 2 * (with_adapter * (K + 2 * N) + used * (P * K + N)), "flops": flops}


# ---------------------------------------------------------------------------
# the operators by their definition, in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    st = prepare(case, seed)
    return _exact_logprobs(st) if case["op"] == "logprobs" else _exact_add(st)


def _exact_add(st):
    y, R = st["y"].double(), st["b"].shape[2]
    for l in range(st["L"]):
        rows = (st["row_ids"] == l).nonzero()[:, 0]
        r = int(st["rank"][l])
        n0 = 0
        for p, n in enumerate(st["parts"]):
            low = st["x"][rows].double() @ st["a"][l, p * R:p * R + r].double().T
            y[rows, n0:n0 + n] += float(st["scale"][l]) * (low @ st["b"][l, n0:n0 + n, :r].double().T)
            n0 += n
    return y


def _exact_logprobs(st):
    x, tokens, top = st["x"], st["tokens"], st["top"]
    T, V = x.shape
    step = max(1, (1 << 27) // V)
    logprobs, entropy, best = [], [], []
    for lo in range(0, T, step):
        rows = torch.log_softmax(x[lo:lo + step].double(), 1)
        p = rows.exp()
        entropy.append(-(p * rows.nan_to_num(neginf=0.0)).sum(1))
        t = tokens[lo:lo + step]
        logprobs.append(torch.where(t >= 0, rows[torch.arange(len(rows), device=x.device), t.clamp(min=0)], 0.0))
        if top:
            best.append(torch.sort(rows, 1, descending=True).values[:, :top])
    out = {"logprobs": torch.cat(logprobs), "entropy": torch.cat(entropy)}
    return out | {"top_ids": None, "top_logprobs": torch.cat(best)} if top else out
