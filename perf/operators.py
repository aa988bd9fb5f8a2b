"""The serving operators for many samples of one prompt, as cases that can be timed and compared.

Three operators belong together when many sequences continue one long prompt: attention that reads
the shared prefix once for all of its sequences (``prefix_attention``), the draw of each sequence's
next token from its filtered distribution (``sample_logits``), and the copies of cache pages that
forking and compacting sequences ask for (``copy_kv_blocks``). ``run`` computes one pass, in plain
torch operations, or (``own``) through this repository's kernels.
"""

import importlib
import math

import numpy as np
import torch

own = False

PACKAGE = "inference-engine-from-scratch_b200"
BLOCK = 16  # tokens in one page of the cache
HEAD = 128  # head dimension


def _ops():
    return importlib.import_module(PACKAGE + ".ops")


# ---------------------------------------------------------------------------------------- cases
def listed():
    attention = [
        # a few users of one short system prompt, one token each: a call whose latency counts
        dict(name="prefix_small", seqs=4, rows=1, ragged=False, heads=16, kv_heads=8, groups=1, prefix=512,
             suffix=48, int8=False),
        # 64 chat users on one system prompt, speculative steps of k = 4 guesses
        dict(name="prefix_chat", seqs=64, rows=5, ragged=True, heads=16, kv_heads=8, groups=1, prefix=2048,
             suffix=300, int8=False),
        # the 8B shape's heads over a long shared document
        dict(name="prefix_document", seqs=64, rows=5, ragged=False, heads=32, kv_heads=8, groups=1, prefix=16384,
             suffix=400, int8=False),
        # the largest batch, one prompt
        dict(name="prefix_batch", seqs=256, rows=5, ragged=True, heads=16, kv_heads=8, groups=1, prefix=4096,
             suffix=200, int8=False),
        # several prompts of different lengths in one batch, some sequences on their own, int8 cache
        dict(name="prefix_groups_int8", seqs=48, rows=5, ragged=True, heads=16, kv_heads=8, groups=6, prefix=3008,
             suffix=160, int8=True),
    ]
    sampling = [
        # one user's next token
        dict(name="sample_one", rows=1, vocab=151936, wide=False, plain_rows=False),
        # 64 users, one token each
        dict(name="sample_chat", rows=64, vocab=151936, wide=False, plain_rows=False),
        # 64 users' rows of a speculative step, unfiltered rows among them
        dict(name="sample_step", rows=320, vocab=151936, wide=False, plain_rows=True),
        # 32-bit logits over an odd vocabulary
        dict(name="sample_fp32_odd", rows=33, vocab=50021, wide=True, plain_rows=True),
    ]
    pages = [
        # one request forked four ways: the pages of its last, partly filled block
        dict(name="pages_fork", layers=28, kv_heads=8, blocks=64, pairs=4, fork=True, int8=False),
        # the pool compacted after many requests have left
        dict(name="pages_compact", layers=28, kv_heads=8, blocks=1024, pairs=400, fork=False, int8=False),
        # the same for an int8 pool of the 8B shape's depth, forked 63 ways
        dict(name="pages_fork_int8", layers=36, kv_heads=8, blocks=256, pairs=63, fork=True, int8=True),
    ]
    return attention + sampling + pages


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "sampling", "sampling", "pages"])
    if kind == "attention":
        while True:
            heads, kv_heads = rng.choice([(16, 8), (32, 8), (4, 2), (8, 1), (8, 8), (14, 2), (20, 4)])
            seqs = _log_uniform(rng, 1, 256)
            rows = rng.choice([1, 2, 5, 5, 9, 17, 40])
            case = dict(seqs=seqs, rows=rows, ragged=rng.random() < 0.7, heads=heads, kv_heads=kv_heads,
                        groups=min(seqs, _log_uniform(rng, 1, 9)), prefix=BLOCK * _log_uniform(rng, 1, 1000),
                        suffix=_log_uniform(rng, 1, 600), int8=rng.random() < 0.35)
            context = case["prefix"] + case["suffix"] + rows
            # neither the work nor the plain form's gathered keys above the largest listed case's
            if work(case)["flops"] <= 8e10 and seqs * context * kv_heads <= 64 * 16800 * 8:
                return case
    if kind == "sampling":
        while True:
            case = dict(rows=_log_uniform(rng, 1, 512), vocab=_log_uniform(rng, 100, 160000),
                        wide=rng.random() < 0.4, plain_rows=rng.random() < 0.5)
            if case["rows"] * case["vocab"] <= 320 * 151936:
                return case
    while True:
        fork = rng.random() < 0.5
        blocks = _log_uniform(rng, 8, 1024)
        case = dict(layers=rng.randint(1, 36), kv_heads=rng.choice([1, 2, 4, 8]), blocks=blocks,
                    pairs=_log_uniform(rng, 1, max(1, blocks // 2 - 1)), fork=fork, int8=rng.random() < 0.4)
        if case["layers"] * case["kv_heads"] * blocks <= 28 * 8 * 1024:
            return case


def _kind(case):
    return "attention" if "prefix" in case else "sampling" if "vocab" in case else "pages"


# ------------------------------------------------------------------------------- attention inputs
def _attention_plan(case):
    """Row counts, contexts, groups and prefix lengths of the batch, from the case alone (so that
    ``work`` counts what every seed's inputs hold)."""
    n = case["seqs"]
    rng = np.random.RandomState(17 + n + case["prefix"] + case["rows"])
    q_len = rng.randint(1, case["rows"] + 1, n) if case["ragged"] else np.full(n, case["rows"])
    suffix = rng.randint(0, case["suffix"] + 1, n)  # tokens after the prefix and before this step's rows
    groups = case["groups"]
    blocks = case["prefix"] // BLOCK
    prefix_blocks = np.array([max(1, blocks * (groups - g) // groups) for g in range(groups)])
    entry_group = np.arange(n) % groups
    rng.shuffle(entry_group)
    if groups > 1:  # every eighth sequence has no shared prefix
        entry_group[::8] = -1
    own_blocks = np.where(entry_group >= 0, prefix_blocks[np.maximum(entry_group, 0)], 0)
    context = own_blocks * BLOCK + suffix + q_len
    return q_len, suffix, entry_group, prefix_blocks, context


def _prepare_attention(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    q_len, _, entry_group, prefix_blocks, context = _attention_plan(case)
    n, nkv = case["seqs"], case["kv_heads"]
    total = -(-context // BLOCK)
    shared = np.where(entry_group >= 0, prefix_blocks[np.maximum(entry_group, 0)], 0)
    used = int(prefix_blocks.sum() + (total - shared).sum())
    num_blocks = used + 3
    ids = np.random.RandomState(seed % (1 << 31)).permutation(num_blocks)[:used]
    group_ids = np.split(ids[: prefix_blocks.sum()], np.cumsum(prefix_blocks)[:-1])
    stride = int(total.max()) + 1
    tables = np.full((n, stride), -1, dtype=np.int32)
    at = int(prefix_blocks.sum())
    for b in range(n):
        s = int(shared[b])
        if s:
            tables[b, :s] = group_ids[entry_group[b]]
        tables[b, s: total[b]] = ids[at: at + total[b] - s]
        at += int(total[b]) - s
    q_start = np.concatenate([[0], np.cumsum(q_len)[:-1]])
    positions = np.concatenate([np.arange(c - q, c) for c, q in zip(context, q_len)])
    slots = num_blocks * BLOCK + 1

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    rows = int(q_len.sum())
    # normalised queries and keys have a spread of scores of a few units; values are about one
    state = dict(case=case, q=(normal(rows, case["heads"], HEAD) * 2.0).to(torch.bfloat16), tables=ints(tables),
                 q_start=ints(q_start), q_len=ints(q_len), positions=ints(positions), entry_group=ints(entry_group),
                 prefix_blocks=ints(prefix_blocks), max_q_len=int(q_len.max()), max_context=int(context.max()),
                 max_prefix=int(prefix_blocks.max()) * BLOCK, k_scale=None, v_scale=None,
                 entry_of=ints(np.repeat(np.arange(n), q_len)))
    if case["int8"]:
        for name in ("k", "v"):
            state[name] = torch.randint(-127, 128, (slots, nkv, HEAD), generator=gen, device=dev, dtype=torch.int8)
            scale = (torch.rand((slots, nkv), generator=gen, device=dev) + 0.5) / 73.0
            state[name + "_scale"] = scale.to(torch.bfloat16)
    else:
        state["k"] = normal(slots, nkv, HEAD).to(torch.bfloat16)
        state["v"] = normal(slots, nkv, HEAD).to(torch.bfloat16)
    return state


def _run_attention(s):
    if own:
        if "workspace" not in s:  # kept by the program, as its other buffers are
            s["workspace"] = _ops().prefix_attention_workspace(
                s["q"].shape[0], s["q_len"].numel(), s["prefix_blocks"].numel(), s["q"].shape[1], s["k"].shape[1],
                s["max_q_len"], s["max_context"], s["q"].device)
            s["out"] = torch.empty_like(s["q"])
        return _ops().prefix_attention(
            s["q"], s["k"], s["v"], s["tables"], s["q_start"], s["q_len"], s["positions"], s["entry_group"],
            s["prefix_blocks"], max_q_len=s["max_q_len"], max_context=s["max_context"], max_prefix=s["max_prefix"],
            k_scale=s["k_scale"], v_scale=s["v_scale"], out=s["out"], workspace=s["workspace"])
    case, dev = s["case"], s["q"].device
    n, nkv = case["seqs"], case["kv_heads"]
    group = case["heads"] // nkv
    # each sequence's keys and values, gathered through its table
    token = torch.arange(s["max_context"], device=dev)
    slot = s["tables"][:, token // BLOCK].long() * BLOCK + token % BLOCK
    slot = torch.where(s["tables"][:, token // BLOCK] >= 0, slot, 0)
    keys, values = s["k"][slot].float(), s["v"][slot].float()
    if s["k_scale"] is not None:
        keys = keys * s["k_scale"][slot].float()[..., None]
        values = values * s["v_scale"][slot].float()[..., None]
    # the rows of each sequence, padded to the longest
    lane = torch.arange(s["max_q_len"], device=dev)
    row = s["q_start"].long()[:, None] + lane
    live = lane < s["q_len"][:, None]
    row = torch.where(live, row, 0)
    q = s["q"][row].float().view(n, s["max_q_len"], nkv, group, HEAD).permute(0, 2, 1, 3, 4)
    q = q.reshape(n, nkv, s["max_q_len"] * group, HEAD)
    scores = torch.matmul(q, keys.permute(0, 2, 3, 1)) / math.sqrt(HEAD)
    seen = token <= torch.where(live, s["positions"][row].long(), -1)[..., None]  # [n, rows, tokens]
    seen = seen[:, None, :, None, :].expand(n, 1, s["max_q_len"], group, -1).reshape(n, 1, -1, token.numel())
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    out = torch.matmul(weight, values.permute(0, 2, 1, 3)) / weight.sum(-1, keepdim=True).clamp(min=1e-38)
    out = out.view(n, nkv, s["max_q_len"], group, HEAD).permute(0, 2, 1, 3, 4)
    out = out.reshape(n, s["max_q_len"], case["heads"], HEAD)
    entry = s["entry_of"].long()
    inside = torch.arange(entry.numel(), device=dev) - s["q_start"].long()[entry]
    return out[entry, inside].to(torch.bfloat16)


def _exact_attention(s):
    case = s["case"]
    nkv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    tables, pos = s["tables"].cpu(), s["positions"].cpu()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (first, count) in enumerate(zip(s["q_start"].tolist(), s["q_len"].tolist())):
        context = int(pos[first + count - 1]) + 1
        slots = (tables[b, : -(-context // BLOCK)].long()[:, None] * BLOCK + torch.arange(BLOCK)).reshape(-1)[:context]
        slots = slots.to(out.device)
        limit = pos[first: first + count].to(out.device)
        hidden = torch.arange(context, device=out.device) > limit[:, None, None]
        for h in range(nkv):
            k, v = s["k"][slots, h].double(), s["v"][slots, h].double()
            if s["k_scale"] is not None:
                k = k * s["k_scale"][slots, h].double()[:, None]
                v = v * s["v_scale"][slots, h].double()[:, None]
            q = s["q"][first: first + count, h * group: (h + 1) * group].double()
            p = (q @ k.T * HEAD ** -0.5).masked_fill(hidden, float("-inf")).softmax(-1)
            out[first: first + count, h * group: (h + 1) * group] = p @ v
    return out


# -------------------------------------------------------------------------------- sampling inputs
# (temperature, top_k, top_p, min_p) of the requests in a batch: greedy ones, the usual chat
# settings, a wide one, and (the last two, where the case has them) unfiltered draws
_SETTINGS = [(0.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 50, 1.0, 0.0), (0.8, 0, 0.9, 0.0),
             (1.0, 0, 1.0, 0.05), (1.2, 200, 0.95, 0.02), (1.0, 0, 1.0, 0.0), (1.5, 0, 0.999, 0.0)]


def _prepare_sampling(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    # logits as language models give them: they fall with the logarithm of the rank, some rows
    # sharply and some slowly, with noise of about one, around a level of their own
    rank = torch.argsort(torch.rand((rows, vocab), generator=gen, device=dev), dim=-1).float() + 1.0
    slope = torch.rand((rows, 1), generator=gen, device=dev) * 1.5 + 1.0
    level = torch.rand((rows, 1), generator=gen, device=dev) * 20.0
    logits = level - slope * torch.log(rank) + torch.randn((rows, vocab), generator=gen, device=dev)
    pick = torch.randint(0, len(_SETTINGS) - (0 if case["plain_rows"] else 2), (rows,), generator=gen, device=dev)
    setting = torch.tensor(_SETTINGS, dtype=torch.float64, device=dev)[pick]
    uniform = torch.randint(0, 1 << 24, (rows,), generator=gen, device=dev).float() * 2.0 ** -24
    return dict(case=case, logits=logits if case["wide"] else logits.to(torch.bfloat16), uniform=uniform,
                temperature=setting[:, 0].float(), top_k=setting[:, 1].int(), top_p=setting[:, 2].float(),
                min_p=setting[:, 3].float())


def _run_sampling(s):
    if own:
        return _ops().sample_logits(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    # 64 bits: the cuts and the draw compare sums over the whole vocabulary with a border
    x = s["logits"].double()
    vocab = x.shape[1]
    greedy = s["temperature"] == 0
    temperature = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    weight = torch.exp((order.values - order.values[:, :1]) / temperature)
    place = torch.arange(vocab, device=x.device)
    count = s["top_k"].long()[:, None]
    count = torch.where((count <= 0) | (count > vocab), vocab, count)
    weight = torch.where(place < count, weight, 0.0)
    mass = torch.cumsum(weight, -1)
    top_p = s["top_p"].double()[:, None]
    keep = (place < count) & ((mass - weight < top_p * mass[:, -1:]) | (top_p >= 1)) & (weight >= s["min_p"].double()[:, None])
    keep = torch.where(greedy[:, None], place < 1, keep) | (place < 1)
    weight = torch.where(keep, weight, 0.0)
    by_id = torch.zeros_like(weight).scatter_(1, order.indices, weight)
    mass = torch.cumsum(by_id, -1)
    target = s["uniform"].double()[:, None] * mass[:, -1:]
    token = torch.argmax((mass > target).to(torch.uint8), dim=-1)
    token = torch.where(greedy, order.indices[:, 0], token)
    probability = by_id.gather(1, token[:, None])[:, 0] / mass[:, -1]
    return token.int(), probability.float()


def _exact_sampling(s):
    tokens, probabilities = [], []
    logits, vocab = s["logits"].double().cpu().numpy(), s["logits"].shape[1]
    settings = zip(s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist(),
                   s["uniform"].tolist())
    for x, (temperature, top_k, top_p, min_p, u) in zip(logits, settings):
        if temperature == 0:
            tokens.append(int(np.argmax(x)))
            probabilities.append(1.0)
            continue
        ranked = np.lexsort((np.arange(vocab), -x))
        if 0 < top_k < vocab:
            ranked = ranked[:top_k]
        w = np.exp((x[ranked] - x.max()) / temperature)
        kept = len(ranked)
        if top_p < 1:
            kept = min(kept, 1 + int(np.searchsorted(np.cumsum(w), top_p * w.sum(), side="left")))
        kept = max(1, min(kept, int((w >= min_p).sum())))
        ids = np.sort(ranked[:kept])
        p = np.exp((x[ids] - x.max()) / temperature)
        below = np.cumsum(p)
        at = min(int(np.searchsorted(below, u * below[-1], side="right")), kept - 1)
        tokens.append(int(ids[at]))
        probabilities.append(float(p[at] / below[-1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probabilities, dtype=torch.float64)


# ----------------------------------------------------------------------------------- page inputs
def _prepare_pages(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    slots = case["blocks"] * BLOCK + 1
    shape = (case["layers"], 2, slots, case["kv_heads"], HEAD)
    scales = None
    if case["int8"]:
        kv = torch.randint(-127, 128, shape, generator=gen, device=dev, dtype=torch.int8)
        scales = torch.rand(shape[:-1], generator=gen, device=dev).to(torch.bfloat16)
    else:
        kv = torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=gen)
    ids = torch.randperm(case["blocks"], generator=gen, device=dev).int()
    pairs = case["pairs"]
    # a fork copies one page to many; compaction moves each page to a place of its own
    src = ids[:1].expand(pairs).contiguous() if case["fork"] else ids[:pairs].contiguous()
    dst = ids[pairs: 2 * pairs].contiguous()
    return dict(case=case, kv=kv, scales=scales, src=src, dst=dst)


def _run_pages(s):
    if own:
        _ops().copy_kv_blocks(s["kv"], s["src"], s["dst"], scales=s["scales"])
        return [s["kv"]] if s["scales"] is None else [s["kv"], s["scales"]]
    inside = torch.arange(BLOCK, device=s["kv"].device)
    src = (s["src"].long()[:, None] * BLOCK + inside).reshape(-1)
    dst = (s["dst"].long()[:, None] * BLOCK + inside).reshape(-1)
    s["kv"][:, :, dst] = s["kv"][:, :, src]
    if s["scales"] is None:
        return [s["kv"]]
    s["scales"][:, :, dst] = s["scales"][:, :, src]
    return [s["kv"], s["scales"]]


# ------------------------------------------------------------------------------------- interface
def prepare(case, seed):
    return {"attention": _prepare_attention, "sampling": _prepare_sampling, "pages": _prepare_pages}[_kind(case)](case, seed)


def run(state):
    return {"attention": _run_attention, "sampling": _run_sampling, "pages": _run_pages}[_kind(state["case"])](state)


def work(case):
    kind = _kind(case)
    if kind == "attention":
        q_len, _, entry_group, prefix_blocks, context = _attention_plan(case)
        shared = np.where(entry_group >= 0, prefix_blocks[np.maximum(entry_group, 0)], 0) * BLOCK
        used = np.unique(entry_group[entry_group >= 0])
        tokens = int(prefix_blocks[used].sum() * BLOCK + (context - shared).sum())
        per_token = 2 * case["kv_heads"] * ((HEAD + 2) if case["int8"] else 2 * HEAD)
        rows = int(q_len.sum())
        # a row at position p reads p + 1 keys; two products of 128 multiply-adds each
        seen = sum(int(q) * int(c) - int(q) * (int(q) - 1) // 2 for q, c in zip(q_len, context))
        return {"bytes": tokens * per_token + 2 * rows * case["heads"] * HEAD * 2,
                "flops": 4.0 * HEAD * case["heads"] * seen}
    if kind == "sampling":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * (4 if case["wide"] else 2) + case["rows"] * 28, "flops": 2.0 * values}
    page = 2 * case["layers"] * BLOCK * case["kv_heads"] * ((HEAD + 2) if case["int8"] else 2 * HEAD)
    return {"bytes": page * ((1 if case["fork"] else case["pairs"]) + case["pairs"]), "flops": 0}


def exact(case, seed):
    kind = _kind(case)
    state = prepare(case, seed)
    if kind == "attention":
        return _exact_attention(state)
    if kind == "sampling":
        return _exact_sampling(state)
    return None  # a copy computes no number
