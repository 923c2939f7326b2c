"""What the operators around drafted tokens, shared prompts and sampled answers are timed on.

Four operators, each through its face in yalm_amd.ops.kernels:
  sample   the next token of every row of logits under its request's own temperature, top-k, top-p and min-p, from
           given uniform numbers (sample_filtered)
  tree     attention of drafted tokens, a tree of them a sequence, over the paged cache that holds the sequence's
           keys and values and theirs (attn_tree)
  fork     whole pages of keys and values copied for sequences that go on from one prompt (copy_pages)
  keep     the drafted tokens that were taken move together behind the sequence's tokens, the others are left behind
           (compact_lines)

A request decodes by these in turn: a step over the drafted tokens (tree), a token for every one of them (sample), and
the lines of the path that was taken moved together (keep); several answers to one prompt begin with fork.

The heads, widths of vocabularies and contexts are those of perf/cases.py, bench.py and the tests: 32 heads of 128 over
8, 24 over 8, the small shape's 4 over 2; vocabularies of 32,000 and 128,256."""
import math

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    """sample: rows, vocab; temperature, top_k, top_p, min_p for all rows, or mixed: every row its own.
    tree: batch, context (tokens held before the drafted ones), nodes; spread: a sequence has down to (1 - spread) of that
    many of either; window 0: every key.  fork, keep: lines (layers) of a cache; pages copied; batch sequences of nodes drafted
    tokens of which kept are taken."""
    return [
        # one chat user's next token under the usual settings: the smallest call, all latency
        dict(name="sample_b1", kind="sample", rows=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0, mixed=False),
        # eight users, the wide vocabulary, a nucleus without a rank
        dict(name="sample_b8_nucleus", kind="sample", rows=8, vocab=128256, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, mixed=False),
        # a full server, or the nodes of eight trees of 32: every row with its request's own settings
        dict(name="sample_b256_mixed", kind="sample", rows=256, vocab=128256, temperature=1.0, top_k=50, top_p=0.95, min_p=0.05, mixed=True),
        # a few drafted tokens on the small model, in float32
        dict(name="tree_small_fp32", kind="tree", dtype="fp32", heads=4, kv_heads=2, head_dim=128, batch=3, context=20, nodes=6, spread=0.9, window=0),
        # one chat user in the middle of a long answer
        dict(name="tree_b1", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, batch=1, context=3056, nodes=16, spread=0.0, window=0),
        # one reader of a long document, a full tree
        dict(name="tree_b1_long", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, batch=1, context=28000, nodes=61, spread=0.0, window=0),
        # four texts beyond the window of a model that keeps one
        dict(name="tree_b4_window", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, batch=4, context=6000, nodes=27, spread=0.0, window=4096),
        # a full server whose requests differ in length and in how much was drafted for them
        dict(name="tree_b64_ragged", kind="tree", dtype="bf16", heads=32, kv_heads=8, head_dim=128, batch=64, context=3041, nodes=40, spread=0.65, window=0),
        # a prompt answered eight times: the page that the prompt ends in, once more for each answer
        dict(name="fork_8", kind="fork", dtype="bf16", lines=32, kv_heads=8, head_dim=128, pages=7, one_source=True),
        # twelve prompts answered eight times
        dict(name="fork_96", kind="fork", dtype="bf16", lines=28, kv_heads=8, head_dim=128, pages=96, one_source=False),
        # one user's path of four drafted tokens
        dict(name="keep_b1", kind="keep", dtype="bf16", lines=32, kv_heads=8, head_dim=128, batch=1, nodes=26, kept=4),
        # a full server's paths
        dict(name="keep_b64", kind="keep", dtype="bf16", lines=32, kv_heads=8, head_dim=128, batch=64, nodes=40, kept=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same kinds over their ranges."""
    kind = rng.choice(["sample", "sample", "tree", "tree", "tree", "fork", "keep"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (24, 8, 128), (4, 2, 128), (32, 8, 64), (16, 16, 64),
                                            (8, 1, 96), (12, 4, 80)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "sample":
        vocab = rng.choice([32000, 32000, 128256, 128256, _log(rng, 300, 128256)])
        return dict(kind=kind, rows=_log(rng, 1, 256), vocab=vocab, temperature=round(rng.uniform(0.3, 1.5), 2),
                    top_k=rng.choice([0, 1, 20, 50, _log(rng, 2, vocab)]), top_p=rng.choice([1.0, 0.95, round(rng.uniform(0.1, 0.99), 2)]),
                    min_p=rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.001, 0.3), 3)]), mixed=rng.random() < 0.4)
    if kind == "tree":
        nodes = rng.choice([_log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 32, 128)])
        batch = _log(rng, 1, 64)
        context = _log(rng, 1, min(28000, 130000 // batch))
        if dtype == "fp32":              # the float32 path serves few sequences
            batch, context = min(batch, 8), min(context, 4000)
        return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, context=context,
                    nodes=min(nodes, max(1, 1700 // batch), max(1, 3400000 // (batch * context))), spread=rng.choice([0.0, round(rng.uniform(0.05, 0.95), 2)]),
                    window=rng.choice([0, 0, 0, _log(rng, 256, 4096)]))
    if kind == "fork":
        return dict(kind=kind, dtype=dtype, lines=rng.randint(2, 24), kv_heads=kv_heads, head_dim=head_dim, pages=_log(rng, 1, 48),
                    one_source=rng.random() < 0.5)
    nodes = rng.randint(2, 64)
    return dict(kind=kind, dtype=dtype, lines=rng.randint(2, 28), kv_heads=kv_heads, head_dim=head_dim, batch=_log(rng, 1, 48),
                nodes=nodes, kept=rng.randint(1, min(nodes, 10 if dtype == "bf16" else 5)))


# ------------------------------------------------------------------------------------------------ what a user has in hand
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _lengths(g, n, most, spread):
    """n lengths from (1 - spread) of most up to it, the first the longest."""
    least = max(1, int(round(most * (1.0 - spread))))
    out = torch.randint(least, most + 1, (n,), generator=g).tolist()
    out[0] = most
    return out


def _trees(g, counts):
    """A tree for each sequence: its nodes in an order in which a parent stands in front of its children, node 0 the root.
    Returns each node's depth and the set of drafted tokens that it sees (itself and its ancestors) as words of 64 bits."""
    words = (max(counts) + 63) // 64
    depths, masks = [], []
    for n in counts:
        depth, mask = [0], [1]
        for i in range(1, n):
            back = int(torch.randint(1, 1 + min(i, 8), (1,), generator=g))
            parent = i - back
            depth.append(depth[parent] + 1)
            mask.append(mask[parent] | (1 << i))
        depths += depth
        for m in mask:
            row = [(m >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
            masks.append([v - (1 << 64) if v >= 1 << 63 else v for v in row])
    return depths, torch.tensor(masks, dtype=torch.int64, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(shape, dtype):
        return torch.randn(shape, generator=gd, device=DEVICE, dtype=torch.float32 if dtype == torch.float32 else dtype)

    kind = case["kind"]
    state = dict(case)
    if kind == "sample":
        R, V = case["rows"], case["vocab"]
        # most tokens far below a few that stand out, more so in some rows than in others
        logits = torch.randn((R, V), generator=gd, device=DEVICE) * 2.5
        lift = 4.0 + 10.0 * torch.rand((R, 1), generator=gd, device=DEVICE)
        at = torch.randint(0, V, (R, 24), generator=gd, device=DEVICE)
        logits.scatter_(1, at, lift * torch.rand((R, 24), generator=gd, device=DEVICE) ** 0.5 + 2.0)
        state["logits"] = logits
        state["u"] = torch.rand(R, generator=gd, device=DEVICE)
        t = torch.full((R,), case["temperature"])
        k = torch.full((R,), case["top_k"], dtype=torch.int32)
        p = torch.full((R,), case["top_p"])
        m = torch.full((R,), case["min_p"])
        if case["mixed"]:                # a third of the rows goes without each of the filters, an eighth is greedy
            t = torch.where(torch.rand(R, generator=g) < 0.125, torch.zeros(R), t * (0.5 + torch.rand(R, generator=g)))
            k = torch.where(torch.rand(R, generator=g) < 0.33, torch.zeros_like(k), k)
            p = torch.where(torch.rand(R, generator=g) < 0.33, torch.ones(R), p)
            m = torch.where(torch.rand(R, generator=g) < 0.33, torch.zeros(R), m)
        state.update(temperature=t.to(DEVICE), top_k=k.to(DEVICE), top_p=p.to(DEVICE), min_p=m.to(DEVICE),
                     out=torch.empty(R, dtype=torch.int32, device=DEVICE), prob=torch.empty(R, device=DEVICE))
        return state
    dt, H, hd = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    state["dtype"] = dt
    if kind == "tree":
        B, window = case["batch"], case["window"]
        held = _lengths(g, B, case["context"], case["spread"])
        counts = _lengths(torch.Generator().manual_seed(B), B, case["nodes"], case["spread"])     # the case's, whatever the seed
        lens = [h + n for h, n in zip(held, counts)]
        pages = [(n + PAGE - 1) // PAGE for n in lens]
        ring = max(pages)
        if window:                       # a windowed cache keeps a ring of pages, with room for the drafted tokens
            ring = min(ring, (window + max(counts) + PAGE - 1) // PAGE + 1)
        n_slots = B + 2
        slots = torch.randperm(n_slots, generator=g)[:B]
        n_pages = sum(min(p, ring) for p in pages) + 1
        free = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((n_slots, ring), -1, dtype=torch.int32)
        for s, p in zip(slots.tolist(), pages):
            for c in range(min(p, ring)):
                table[s, c] = free.pop()
        depths, mask = _trees(g, counts)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        base = torch.tensor(held).repeat_interleave(torch.tensor(counts))
        state.update(q=normal((cu[-1], case["heads"] * hd), dt), k_pages=normal((n_pages, H, PAGE, hd), dt),
                     v_pages=normal((n_pages, H, hd, PAGE), dt), table=table.to(DEVICE), ring=ring, seq_slot=_i32(slots.tolist()),
                     seq_len=_i32(lens), cu_nodes=_i32(cu), mask=mask, positions=_i32((base + torch.tensor(depths)).tolist()),
                     step_max_len=_i32([max(lens)]), max_nodes=max(counts), max_len=max(lens), out=torch.empty((cu[-1], case["heads"] * hd), dtype=dt, device=DEVICE))
        return state
    L = case["lines"]
    if kind == "fork":
        n = case["pages"]
        n_pages = 2 * n + 3
        order = torch.randperm(n_pages, generator=g)
        src = order[:1].repeat(n) if case["one_source"] else order[:n]
        state.update(src=src.to(torch.int32).to(DEVICE), dst=order[n + 1:2 * n + 1].to(torch.int32).to(DEVICE))
    else:
        B, nodes, kept = case["batch"], case["nodes"], case["kept"]
        n_slots, columns = B + 1, 4
        n_pages = n_slots * columns
        order = torch.randperm(n_pages, generator=g)
        slots = torch.randperm(n_slots, generator=g)[:B].tolist()
        start = torch.randint(1, PAGE * columns - nodes, (B,), generator=g).tolist()
        keep, cu = [], [0]
        for _ in range(B):
            # a path: the root, and deeper nodes, which stand behind more nodes than the path has in front of them
            k = 1 + int(torch.randint(0, kept, (1,), generator=g)) if B > 1 else kept
            deeper = (k + torch.randperm(nodes - k, generator=g)[:k - 1]).sort().values.tolist()
            keep += [0] + deeper
            cu.append(len(keep))
        state.update(table=order.view(n_slots, columns).to(torch.int32).to(DEVICE), ring=columns, seq_slot=_i32(slots), start=_i32(start),
                     keep=_i32(keep), cu_keep=_i32(cu), max_keep=max(b - a for a, b in zip(cu, cu[1:])))
    state.update(k_pages=normal((L, n_pages, H, PAGE, hd), dt), v_pages=normal((L, n_pages, H, hd, PAGE), dt))
    return state


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_sample(s):
    x, V = s["logits"], s["logits"].shape[1]
    greedy = ~(s["temperature"] > 0)
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    ranked, order = x.sort(dim=1, descending=True, stable=True)
    z = ranked.double()
    w = torch.exp((z - z[:, :1]) / t)
    rank = torch.arange(V, device=x.device)[None, :]
    k = s["top_k"].long()[:, None]
    k = torch.where(k > 0, k, torch.full_like(k, V))
    k = torch.where(greedy[:, None], torch.ones_like(k), k)
    w = torch.where(rank < k, w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    p = s["top_p"].double()[:, None]
    in_p = (before < p * w.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)
    taken = in_p & (w > 0) & ((w >= s["min_p"].double()[:, None]) | (rank == 0))
    w = torch.where(taken, w, torch.zeros_like(w))
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    total = by_index.sum(1, keepdim=True)
    reached = (by_index.cumsum(1) >= s["u"].double()[:, None] * total) & (by_index > 0)
    last = V - 1 - (by_index > 0).flip(1).to(torch.int32).argmax(1)
    token = torch.where(reached.any(1), reached.to(torch.int32).argmax(1), last)
    prob = by_index.gather(1, token[:, None])[:, 0] / total[:, 0]
    return {"token": token.to(torch.int32), "prob": prob.float()}


def _row_places(head_dim):
    """How keys and values lie inside a page of a head: keys [row][element] and values [element][row], or with heads that are
    multiples of 32 in blocks: keys [element / 32][place of the row][element % 32], values [row / 32][element][row % 32]."""
    r = torch.arange(PAGE, device=DEVICE)
    return head_dim % 32 == 0, 16 * (2 * (r // 32) + (r // 4) % 2) + 4 * ((r // 8) % 4) + r % 4


def _rows_of(k, v, head_dim):
    """Pages [..., 64, hd] of keys and [..., hd, 64] of values as rows [..., 64, hd] both."""
    blocks, place = _row_places(head_dim)
    lead = k.shape[:-2]
    if not blocks:
        return k, v.transpose(-1, -2)
    k = k.reshape(lead + (head_dim // 32, PAGE, 32)).index_select(len(lead) + 1, place)
    v = v.reshape(lead + (2, head_dim, 32))
    return k.transpose(-3, -2).reshape(lead + (PAGE, head_dim)), v.transpose(-1, -2).reshape(lead + (PAGE, head_dim))


def _plain_tree(s):
    nh, H, hd, window = s["heads"], s["kv_heads"], s["head_dim"], s["window"]
    G, N, B = nh // H, s["max_nodes"], s["seq_len"].shape[0]
    cu = s["cu_nodes"].long()
    count = cu[1:] - cu[:-1]
    lens = s["seq_len"].long()
    base = lens - count
    # the pages that any of a sequence's drafted tokens sees
    first = (base - window + 1).clamp_min(0) // PAGE if window else torch.zeros_like(base)
    most = min(s["ring"], s["table"].shape[1])
    page = first[:, None] + torch.arange(most, device=DEVICE)[None, :]
    phys = s["table"].long()[s["seq_slot"].long()].gather(1, page % s["ring"]).clamp_min(0)
    k, v = _rows_of(s["k_pages"][phys], s["v_pages"][phys], hd)              # [B, pages, H, 64, hd]
    pos = (page[:, :, None] * PAGE + torch.arange(PAGE, device=DEVICE)).reshape(B, -1)
    there = pos < lens[:, None]
    L = pos.shape[1]
    k = k.transpose(1, 2).reshape(B, H, L, hd).float().masked_fill(~there[:, None, :, None], 0.0)
    v = v.transpose(1, 2).reshape(B, H, L, hd).float().masked_fill(~there[:, None, :, None], 0.0)
    row = (cu[:-1, None] + torch.arange(N, device=DEVICE)).clamp_max(s["q"].shape[0] - 1)
    live = torch.arange(N, device=DEVICE)[None, :] < count[:, None]
    q = s["q"][row].float().view(B, N, H, G, hd).permute(0, 2, 3, 1, 4).reshape(B, H, G * N, hd)
    # who sees what: a key of the sequence by the window, a drafted one by the tree
    node = (pos - base[:, None]).clamp(0, 64 * s["mask"].shape[1] - 1)
    word = s["mask"][row].gather(2, (node // 64)[:, None, :].expand(B, N, L))
    drafted = ((word >> (node % 64)[:, None, :]) & 1) != 0
    held = torch.ones_like(drafted)
    if window:
        held = pos[:, None, :] > s["positions"].long()[row][:, :, None] - window
    sees = torch.where((pos >= base[:, None])[:, None, :], drafted, held) & there[:, None, :] & live[:, :, None]
    score = (q @ k.transpose(-1, -2)).view(B, H, G, N, L) * (1.0 / math.sqrt(hd))
    score = score.masked_fill(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = (e.view(B, H, G * N, L) @ v).view(B, H, G, N, hd) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, nh * hd)
    out = torch.empty_like(s["q"])
    out[row[live]] = o[live].to(out.dtype)
    return out


def _plain_fork(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_keep(s):
    hd = s["head_dim"]
    blocks, place = _row_places(hd)
    cu = s["cu_keep"].long()
    n = s["keep"].shape[0]
    seq = torch.searchsorted(cu, torch.arange(n, device=DEVICE), right=True) - 1
    begin = s["start"].long()[seq]
    src, dst = begin + s["keep"].long(), begin + torch.arange(n, device=DEVICE) - cu[seq]
    rows = s["table"].long()[s["seq_slot"].long()[seq]]
    e = torch.arange(hd, device=DEVICE)[None, :]

    def where(pos):
        page = rows.gather(1, (pos // PAGE % s["ring"])[:, None])
        r = (pos % PAGE)[:, None]
        if blocks:
            return page, ((e // 32) * PAGE + place[r]) * 32 + e % 32, ((r // 32) * hd + e) * 32 + r % 32
        return page, r * hd + e, e * PAGE + r

    (p0, k0, v0), (p1, k1, v1) = where(src), where(dst)
    k = s["k_pages"].view(s["k_pages"].shape[:3] + (-1,))
    v = s["v_pages"].view(s["v_pages"].shape[:3] + (-1,))
    k[:, p1, :, k1] = k[:, p0, :, k0]
    v[:, p1, :, v1] = v[:, p0, :, v0]
    return {"k": s["k_pages"], "v": s["v_pages"]}


# ------------------------------------------------------------------------------------------------ one pass
def _own_sample(s):
    from yalm_amd.ops import kernels
    ws = s.get("workspace")
    if ws is None:
        ws = s["workspace"] = torch.zeros(kernels.sample_filtered_workspace(s["rows"], s["vocab"]), dtype=torch.int32, device=DEVICE)
    kernels.sample_filtered(s["logits"], s["u"], s["out"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                            min_p=s["min_p"], prob=s["prob"], workspace=ws)
    return {"token": s["out"], "prob": s["prob"]}


def _own_tree(s):
    from yalm_amd.ops import kernels
    nh, H, hd = s["heads"], s["kv_heads"], s["head_dim"]
    plan = s.get("plan")
    if plan is None:
        n_splits = kernels.attn_tree_splits(s["batch"], s["max_nodes"], s["max_len"], nh, H, hd, s["dtype"], s["window"])
        partial = torch.empty(kernels.attn_tree_workspace_floats(s["q"].shape[0], nh, hd, n_splits), device=DEVICE)
        plan = s["plan"] = (n_splits, partial)
    kernels.attn_tree(s["q"], s["k_pages"], s["v_pages"], s["table"], s["ring"], s["seq_slot"], s["seq_len"], s["cu_nodes"], s["mask"],
                      s["out"], plan[1], nh, H, hd, s["window"], plan[0], s["max_nodes"], positions=s["positions"], step_max_len=s["step_max_len"])
    return s["out"]


def _own_fork(s):
    from yalm_amd.ops import kernels
    kernels.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _own_keep(s):
    from yalm_amd.ops import kernels
    kernels.compact_lines(s["k_pages"], s["v_pages"], s["table"], s["ring"], s["seq_slot"], s["start"], s["cu_keep"], s["keep"], s["max_keep"])
    return {"k": s["k_pages"], "v": s["v_pages"]}


_PLAIN = {"sample": _plain_sample, "tree": _plain_tree, "fork": _plain_fork, "keep": _plain_keep}
_OWN = {"sample": _own_sample, "tree": _own_tree, "fork": _own_fork, "keep": _own_keep}


def run(state):
    if own:
        return _OWN[state["kind"]](state)
    return _PLAIN[state["kind"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "sample":         # the logits once; a subtraction, an exponential and a sum for each
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 28.0 * case["rows"], "flops": 4.0 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    H, hd = case["kv_heads"], case["head_dim"]
    if case["kind"] == "tree":
        mean = 1.0 - case["spread"] / 2 if case["batch"] > 1 else 1.0
        held, nodes = case["context"] * mean, max(1.0, case["nodes"] * mean)
        keys = min(held, case["window"]) if case["window"] else held
        B, nh = case["batch"], case["heads"]
        return {"bytes": B * (2.0 * (keys + nodes) * H * hd * size + 2.0 * nodes * nh * hd * size),
                "flops": B * 4.0 * nodes * nh * hd * (keys + nodes / 4)}
    if case["kind"] == "fork":
        page = 2.0 * case["lines"] * H * PAGE * hd * size
        return {"bytes": page * (case["pages"] + (1 if case["one_source"] else case["pages"])), "flops": 0.0}
    kept = case["kept"] if case["batch"] == 1 else (case["kept"] + 1) / 2.0
    return {"bytes": 2.0 * 2.0 * max(1.0, case["batch"] * (kept - 1)) * case["lines"] * H * hd * size, "flops": 0.0}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _exact_sample(s):
    """The row in the order of its ranks, each filter as its definition says, and the walk in the order of the tokens."""
    R, V = s["logits"].shape
    tokens, probs = [], []
    for r in range(R):
        x = s["logits"][r].double()
        t = float(s["temperature"][r])
        if not t > 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            probs.append(1.0)
            continue
        p = torch.softmax(x / t, 0)
        order = torch.argsort(x, descending=True, stable=True)
        k = int(s["top_k"][r])
        if k > 0:
            order = order[:k]
        q = p[order] / p[order].sum()
        limit = float(s["top_p"][r])
        if limit < 1:
            n = int((q.cumsum(0) < limit).sum()) + 1
            order = order[:n]
        floor = float(s["min_p"][r]) * float(p.max())
        order = order[(p[order] >= floor) | (torch.arange(order.shape[0], device=order.device) == 0)]
        order = order.sort().values
        c = p[order].cumsum(0)
        at = min(int((c < float(s["u"][r]) * c[-1]).sum()), order.shape[0] - 1)
        tokens.append(int(order[at]))
        probs.append(float(p[order[at]] / c[-1]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}


def _exact_tree(s):
    nh, H, hd, window = s["heads"], s["kv_heads"], s["head_dim"], s["window"]
    cu, lens, slots = s["cu_nodes"].tolist(), s["seq_len"].tolist(), s["seq_slot"].tolist()
    outs = []
    for b, (a, z) in enumerate(zip(cu, cu[1:])):
        n, base = z - a, lens[b] - (z - a)
        first = max(0, base - window + 1) // PAGE if window else 0
        pages = list(range(first, (lens[b] - 1) // PAGE + 1))
        phys = s["table"][slots[b]].long()[torch.tensor([p % s["ring"] for p in pages], device=DEVICE)]
        k, v = _rows_of(s["k_pages"][phys], s["v_pages"][phys], hd)
        lo, hi = first * PAGE, lens[b]
        k = k.transpose(0, 1).reshape(H, -1, hd)[:, :hi - lo].double()
        v = v.transpose(0, 1).reshape(H, -1, hd)[:, :hi - lo].double()
        sees = torch.ones((n, hi - lo), dtype=torch.bool, device=DEVICE)
        if window:
            sees &= torch.arange(lo, hi, device=DEVICE)[None, :] > s["positions"][a:z].long()[:, None] - window
        for j in range(n):               # a drafted token's key: for those whose set names it
            sees[:, base - lo + j] = ((s["mask"][a:z, j // 64] >> (j % 64)) & 1) != 0
        group = nh // H
        o = torch.empty((n, nh, hd), dtype=torch.float64, device=DEVICE)
        for h in range(nh):
            score = s["q"][a:z].view(n, nh, hd)[:, h].double() @ k[h // group].t() / math.sqrt(hd)
            o[:, h] = torch.softmax(score.masked_fill(~sees, -math.inf), -1) @ v[h // group]
        outs.append(o.reshape(n, nh * hd))
    return torch.cat(outs)


def _exact_fork(s):
    k, v = s["k_pages"].double(), s["v_pages"].double()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        k[:, b] = s["k_pages"][:, a].double()
        v[:, b] = s["v_pages"][:, a].double()
    return {"k": k, "v": v}


def _exact_keep(s):
    hd = s["head_dim"]
    blocks, place = _row_places(hd)
    k, v = s["k_pages"].double(), s["v_pages"].double()
    lead = k.shape[:3]
    # a token's key is kr[:, page, :, :, place], its value vr[:, page, :, half, :, row of the half]
    kr, vr = (k.view(lead + (hd // 32, PAGE, 32)), v.view(lead + (2, hd, 32))) if blocks else (k.view(lead + (1, PAGE, hd)), v.view(lead + (1, hd, PAGE)))
    half = vr.shape[-1]
    place = place.tolist() if blocks else list(range(PAGE))
    cu, keep, table = s["cu_keep"].tolist(), s["keep"].tolist(), s["table"].tolist()
    for b, (slot, start) in enumerate(zip(s["seq_slot"].tolist(), s["start"].tolist())):
        moves = [(start + i, start + at) for at, i in enumerate(keep[cu[b]:cu[b + 1]])]
        for source, to in moves:         # ascending: nothing is written before it has been read
            (p0, r0), (p1, r1) = ((table[slot][x // PAGE % s["ring"]], x % PAGE) for x in (source, to))
            kr[:, p1, :, :, place[r1]] = kr[:, p0, :, :, place[r0]].clone()
            vr[:, p1, :, r1 // half, :, r1 % half] = vr[:, p0, :, r0 // half, :, r0 % half].clone()
    return {"k": k, "v": v}


def exact(case, seed):
    return {"sample": _exact_sample, "tree": _exact_tree, "fork": _exact_fork, "keep": _exact_keep}[case["kind"]](prepare(case, seed))
