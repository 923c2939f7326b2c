"""The operators around drafted tokens and sampled answers, each against its definition in 64 bits on the CPU: sampling under
filters from given numbers, attention of trees of drafted tokens over the cache, pages copied and lines moved together, and a
run of them as a drafted step uses them."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kernels import DEV, K, i32, pages_as_rows, pages_as_stored, rnd

pytestmark = pytest.mark.gpu
PAGE = 64


# ------------------------------------------------------------------------------------------------ sampling under filters
def sample_reference(row, u, T=1.0, k=0, p=1.0, mp=0.0):
    """(token, probability) of one row in 64 bits; the settings as the float32 numbers that the kernel is given."""
    T, p, mp, u = (float(np.float32(x)) for x in (T, p, mp, u))
    x = row.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not x.max() > -np.inf:
        return -1, 0.0
    if not T > 0:
        return int(x.argmax()), 1.0
    with np.errstate(invalid="ignore"):
        z = np.where(x == x.max(), 0.0, (x - x.max()) / T)
    w = np.exp(z)
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(order):
        order = order[:k]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        order = order[(before < p * w[order].sum()) | (np.arange(len(order)) == 0)]
    order = np.sort(order[(w[order] >= mp) & (w[order] > 0)])
    c = np.cumsum(w[order])
    at = min(int((c < u * c[-1]).sum()), len(order) - 1)
    return int(order[at]), float(w[order[at]] / c[-1])


def check_sampled(logits, u, out, prob, T, k, p, mp, what=""):
    """Tokens equal; a probability is a float32 rounding (2^-24) of a quotient whose total is off by 2^-45 a token of it."""
    got, gp = out.cpu().numpy(), prob.double().cpu().numpy()
    rows = logits.cpu().numpy()
    for r in range(rows.shape[0]):
        token, want = sample_reference(rows[r], u[r], T[r], k[r], p[r], mp[r])
        assert got[r] == token, (what, r, got[r], token, T[r], k[r], p[r], mp[r], u[r])
        assert abs(gp[r] - want) <= want * (2.0 ** -23 + rows.shape[1] * 2.0 ** -45), (what, r, gp[r], want)


def draw_rows(logits, u, T, k, p, mp):
    n = logits.shape[0]
    dev = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=DEV)  # noqa: E731
    out = torch.full((n,), -7, dtype=torch.int32, device=DEV)
    prob = torch.full((n,), float("nan"), device=DEV)
    x = logits.to(DEV)
    args = dict(temperature=dev(T, torch.float32), top_k=dev(k, torch.int32), top_p=dev(p, torch.float32), min_p=dev(mp, torch.float32))
    # a row a workgroup, and rows over several of them through a workspace that holds anything
    K().sample_filtered(x, dev(u, torch.float32), out, prob=prob, **args)
    ws = torch.randint(-2 ** 31, 2 ** 31 - 1, (K().sample_filtered_workspace(*x.shape),), dtype=torch.int32, device=DEV)
    out2, prob2 = torch.full_like(out, -9), torch.full_like(prob, float("nan"))
    K().sample_filtered(x, dev(u, torch.float32), out2, prob=prob2, workspace=ws, **args)
    assert torch.equal(out, out2) and torch.equal(prob, prob2)
    return out2, prob2


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.3, 0, 0.9, 0.0), (0.5, 0, 1.0, 0.1), (1.0, 1, 1.0, 0.0), (0.7, 300, 0.5, 0.02),
            (1.0, 5, 1e-9, 0.0), (0.0, 7, 0.4, 0.3), (100.0, 0, 0.37, 0.0), (1e-4, 0, 0.99, 0.0), (2.0, 0, 0.999, 1.0), (1.0, 1 << 30, 1.0, 0.0)]


@pytest.mark.parametrize("R", [1, 12, 40])
@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 65, 255, 1023, 4097, 32000, 128256])
def test_filtered_sampling_equals_its_definition(V, R):
    settings = [SETTINGS[(r + V) % len(SETTINGS)] for r in range(R)]
    logits = rnd((R, V), 5 + V, torch.float32, 2.5)
    u = np.random.default_rng(V).random(R).astype(np.float32)
    u[0] = 0.0
    u[-1] = 1.0 - 2.0 ** -24
    T, k, p, mp = (list(x) for x in zip(*settings))
    check_sampled(logits, u, *draw_rows(logits, u, T, k, p, mp), T, k, p, mp, "V %d" % V)


def odd_rows(V, g):
    """Rows on which an order is least what it is elsewhere: equal logits, few values, sorted ones, borders inside equal
    logits, infinities, no numbers, zeros of both signs, values next to each other."""
    inf, nan = float("inf"), float("nan")
    base = torch.randn(V, generator=g) * 2
    rows = {"equal": torch.full((V,), -3.25), "two values": (torch.rand(V, generator=g) < 0.3).float() * 0.0 + torch.where(torch.rand(V, generator=g) < 0.3, 1.0, 0.0),
            "falling": torch.linspace(6, -6, V), "rising": torch.linspace(-6, 6, V), "steps": torch.floor(base * 2) / 2,
            "masked": torch.where(torch.rand(V, generator=g) < 0.9, -inf, 1.0) * 1.0, "lowest": torch.where(torch.rand(V, generator=g) < 0.9, torch.finfo(torch.float32).min, 1.0),
            "nan": torch.where(torch.rand(V, generator=g) < 0.2, nan, 1.0) * base, "zeros": torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0),
            "near": 1.0 + torch.randint(0, 900, (V,), generator=g) * 2.0 ** -23, "one": torch.full((V,), -inf), "inf": base.clone(),
            "huge": base * 1e37, "tiny": base * 1e-38, "wide": base * 40, "big": 1e6 + torch.floor(base)}
    rows["masked"][V // 2] = 0.5
    rows["lowest"][V // 2] = 2.0
    rows["nan"][V - 1] = 0.25
    rows["one"][V - 1] = -1e30
    rows["inf"][[0, V // 3, V - 1]] = inf
    return rows


@pytest.mark.parametrize("V", [7, 300, 5003, 32000])
def test_filtered_sampling_of_odd_rows(V):
    g = torch.Generator().manual_seed(V)
    rows = odd_rows(V, g)
    settings = SETTINGS + [(1.0, V // 2, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, V // 3 + 1, 0.25, 0.0), (0.25, 2, 0.75, 0.0), (1e-30, 0, 0.5, 0.0), (1e30, 0, 0.5, 0.0)]
    for name, row in rows.items():
        logits = row.repeat(len(settings), 1)
        u = np.random.default_rng(V).random(len(settings)).astype(np.float32)
        T, k, p, mp = (list(x) for x in zip(*settings))
        check_sampled(logits, u, *draw_rows(logits, u, T, k, p, mp), T, k, p, mp, name)


FAR = [(1.0, 769, 1.0, 0.0), (0.7, 1000, 0.95, 0.0), (1.0, 768, 0.9, 0.0), (0.6, 4000, 0.3, 0.05), (1.5, 9999, 0.9999, 0.0), (1.0, 800, 1e-9, 0.0),
       (100.0, 2000, 0.5, 0.0), (1e-3, 2000, 0.5, 0.0), (3.0, 1500, 1.0, 0.3), (0.3, 60000, 0.99, 0.0), (1.0, 100000, 1.0, 0.0), (2.0, 20000, 0.75, 0.001)]


@pytest.mark.parametrize("V", [770, 1000, 4097, 32001, 128256])
@pytest.mark.parametrize("width", [0.5, 2.5, 12.0])
def test_ranks_behind_many_tokens(V, width):
    settings = FAR + [(0.9, V - 1, 0.97, 0.0), (0.9, V // 2, 1.0, 0.0)]
    logits = rnd((len(settings), V), V + int(width), torch.float32, width)
    u = np.random.default_rng(V).random(len(settings)).astype(np.float32)
    T, k, p, mp = (list(x) for x in zip(*settings))
    check_sampled(logits, u, *draw_rows(logits, u, T, k, p, mp), T, k, p, mp, "V %d" % V)


@pytest.mark.parametrize("V", [1200, 20011])
def test_ranks_behind_many_tokens_of_odd_rows(V):
    for name, row in odd_rows(V, torch.Generator().manual_seed(V)).items():
        logits = row.repeat(len(FAR), 1)
        u = np.random.default_rng(V).random(len(FAR)).astype(np.float32)
        T, k, p, mp = (list(x) for x in zip(*FAR))
        check_sampled(logits, u, *draw_rows(logits, u, T, k, p, mp), T, k, p, mp, name)


def test_rows_with_nothing_to_draw_and_settings_left_out():
    nothing = torch.stack([torch.full((50,), -float("inf")), torch.full((50,), float("nan"))]).to(DEV)
    out, prob = torch.zeros(2, dtype=torch.int32, device=DEV), torch.ones(2, device=DEV)
    u = torch.tensor([0.3, 0.9], device=DEV)
    K().sample_filtered(nothing, u, out, prob=prob)
    assert out.tolist() == [-1, -1] and prob.tolist() == [0.0, 0.0]
    logits = rnd((2, 999), 3).to(DEV)
    K().sample_filtered(logits, u, out)
    assert out.tolist() == [sample_reference(logits[r].cpu().numpy(), float(u[r]))[0] for r in range(2)]
    K().sample_filtered(logits[:0], u[:0], out[:0])           # no rows: nothing happens


def test_the_share_of_draws_is_the_probability():
    """All multiples of 1 / 4,096 as numbers: each kept token is drawn within two of 4,096 times its share."""
    row = rnd((1, 60), 9, torch.float32, 1.5)
    n = 4096
    u = (np.arange(n) / n).astype(np.float32)
    out, _ = draw_rows(row.repeat(n, 1), u, [0.9] * n, [20] * n, [0.9] * n, [0.01] * n)
    x = np.exp((row[0].double().numpy() - row.max().item()) / float(np.float32(0.9)))
    order = np.argsort(-x)[:20]
    c = np.cumsum(x[order])
    order = order[(c - x[order] < float(np.float32(0.9)) * c[-1])]
    share = np.bincount(out.cpu().numpy(), minlength=60) / n
    want = np.zeros(60)
    want[order] = x[order] / x[order].sum()
    assert np.abs(share - want).max() <= 2.0 / n


def test_filtered_sampling_in_a_graph_and_on_another_stream():
    logits = rnd((9, 5000), 21, torch.float32, 2.0).to(DEV)
    settings = [SETTINGS[i % len(SETTINGS)] for i in range(9)]
    T, k, p, mp = (torch.tensor(x, dtype=torch.int32 if i == 1 else torch.float32, device=DEV) for i, x in enumerate(zip(*settings)))
    u = torch.rand(9, generator=torch.Generator().manual_seed(2)).to(DEV)
    out, prob = torch.zeros(9, dtype=torch.int32, device=DEV), torch.zeros(9, device=DEV)
    ws = torch.zeros(K().sample_filtered_workspace(9, 5000), dtype=torch.int32, device=DEV)

    def go():
        K().sample_filtered(logits, u, out, temperature=T, top_k=k, top_p=p, min_p=mp, prob=prob, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for i in range(4):
        u.copy_(torch.rand(9, generator=torch.Generator().manual_seed(40 + i)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = out.tolist()
        check_sampled(logits, u.cpu().numpy(), out, prob, *(x.cpu().tolist() for x in (T, k, p, mp)), "replay %d" % i)
        go()
        assert out.tolist() == want


# ------------------------------------------------------------------------------------------------ pages and lines that move
@pytest.mark.parametrize("shape,dtype", [((3, 11, 2, 64, 128), torch.bfloat16), ((2, 9, 3, 64, 48), torch.float32), ((1, 7, 1, 64, 6), torch.bfloat16),
                                         ((2, 5, 3), torch.uint8), ((4, 6, 1001), torch.bfloat16), ((2, 300, 5, 7), torch.float32)])
@pytest.mark.parametrize("n", [1, 3, 280])
def test_copied_pages(shape, dtype, n):
    g = torch.Generator().manual_seed(n)
    a = torch.randint(0, 127, shape, generator=g).to(dtype).to(DEV)
    b = torch.randint(0, 127, shape, generator=g).to(dtype).to(DEV)
    pages = shape[1]
    order = torch.randperm(pages, generator=g)
    cut = pages // 2
    src, dst = order[:cut], order[cut:]
    src = src[torch.randint(0, cut, (n,), generator=g)]
    dst = dst[torch.arange(n) % len(dst)]                      # more pairs than pages: the last of a destination stands
    want_a, want_b = a.clone(), b.clone()
    for s, d in zip(src.tolist(), dst.tolist()):
        want_a[:, d], want_b[:, d] = a[:, s], b[:, s]
    one = a.clone()
    K().copy_pages(a, b, src.to(torch.int32).to(DEV), dst.to(torch.int32).to(DEV))
    assert torch.equal(a, want_a) and torch.equal(b, want_b)
    K().copy_pages(one, None, src.to(torch.int32).to(DEV), dst.to(torch.int32).to(DEV))
    assert torch.equal(one, want_a)


def test_copied_pages_pass_over_what_is_no_page_and_copy_none():
    a = torch.arange(24.0, device=DEV).view(2, 4, 3)
    want = a.clone()
    want[:, 2] = a[:, 1]
    K().copy_pages(a, None, i32([1, 0, 9, -1, 0, 4]), i32([2, 7, 3, 3, -5, 2]))
    assert torch.equal(a, want)
    K().copy_pages(a, None, i32([]), i32([]))
    assert torch.equal(a, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,H,ring", [(128, 2, 4), (64, 1, 3), (48, 3, 3), (6, 1, 3), (96, 8, 5), (272, 1, 3), (32, 2, 3), (160, 1, 3), (1024, 1, 3)])
def test_kept_lines_move_together(hd, H, ring, dtype):
    """Paths of every length, the first and the last place of a page, a ring that wraps, a row without a slot; all else stays."""
    g = torch.Generator().manual_seed(hd)
    L, n_slots = 3, 7
    n_pages = n_slots * ring + 1
    kp = torch.randint(-99, 99, (L, n_pages, H, PAGE, hd), generator=g).to(dtype)
    vp = torch.randint(-99, 99, (L, n_pages, H, hd, PAGE), generator=g).to(dtype)
    table = torch.randperm(n_pages, generator=g)[:n_slots * ring].view(n_slots, ring).to(torch.int32)
    # (slot, start, kept nodes): the whole tree, nothing, single ones, long lists over page ends
    seqs = [(3, 60, [0, 2, 3, 9]), (0, 0, list(range(40))), (5, 63, [1]), (1, 64 * ring - 8, [0, 5, 6, 7, 20, 33]), (-1, 5, [0, 4]),
            (6, 1, sorted(torch.randperm(100, generator=g)[:57].tolist())), (4, 127, []), (2, 1000, [0, 63, 64, 65])]
    want_k, want_v = kp.clone(), vp.clone()
    for slot, start, keep in seqs:
        if slot < 0:
            continue
        for i, j in enumerate(keep):
            (p0, r0), (p1, r1) = ((int(table[slot, x // PAGE % ring]), x % PAGE) for x in (start + j, start + i))
            want_k[:, p1, :, r1, :] = want_k[:, p0, :, r0, :].clone()
            want_v[:, p1, :, :, r1] = want_v[:, p0, :, :, r0].clone()
    stored = lambda a, b: tuple(torch.stack(x) for x in zip(*(pages_as_stored(a[i], b[i]) for i in range(L))))  # noqa: E731
    (ks, vs), (wk, wv) = stored(kp, vp), stored(want_k, want_v)
    ks, vs = ks.to(DEV), vs.to(DEV)
    flat, cu = [], [0]
    for _, _, keep in seqs:
        flat += keep
        cu.append(len(flat))
    K().compact_lines(ks, vs, table.to(DEV), ring, i32([s for s, _, _ in seqs]), i32([s for _, s, _ in seqs]), i32(cu), i32(flat),
                      max(len(k) for _, _, k in seqs))
    assert torch.equal(ks.cpu(), wk) and torch.equal(vs.cpu(), wv)


# ------------------------------------------------------------------------------------------------ trees over the cache
def random_tree(n, g, chain=False):
    """[(parent)], depth and the bits of what each node sees."""
    depth, seen = [0], [1]
    for i in range(1, n):
        parent = i - 1 if chain else i - int(torch.randint(1, 1 + min(i, 9), (1,), generator=g))
        depth.append(depth[parent] + 1)
        seen.append(seen[parent] | 1 << i)
    return depth, seen


def words_of(seen, words):
    out = []
    for m in seen:
        row = [(m >> (64 * w)) & ((1 << 64) - 1) for w in range(words)]
        out.append([x - (1 << 64) if x >= 1 << 63 else x for x in row])
    return torch.tensor(out, dtype=torch.int64)


def tree_case(held, nodes, n_heads, n_kv, hd, dtype, window=0, seed=0, words=None, chain=False):
    """Sequences of held[b] tokens and nodes[b] drafted ones in pages; whatever holds no token is NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(held)
    lens = [h + n for h, n in zip(held, nodes)]
    full = max(1, max((n + PAGE - 1) // PAGE for n in lens))
    ring = min(full, (window + max(nodes) + PAGE - 1) // PAGE + 1) if window else full
    n_slots, n_pages = B + 2, B * ring + 2
    kp = torch.full((n_pages, n_kv, PAGE, hd), float("nan"), dtype=dtype)
    vp = torch.full((n_pages, n_kv, hd, PAGE), float("nan"), dtype=dtype)
    order = torch.randperm(n_pages, generator=g).tolist()
    slots = torch.randperm(n_slots, generator=g)[:B].tolist()
    table = torch.full((n_slots, ring), -1, dtype=torch.int32)
    keys, vals, depths, seen = [], [], [], []
    for b, n in enumerate(lens):
        k, v = rnd((n, n_kv, hd), seed + 7 * b, dtype), rnd((n, n_kv, hd), seed + 7 * b + 1, dtype)
        keys.append(k)
        vals.append(v)
        last = (n - 1) // PAGE if n else -1
        for a in range(max(0, last - ring + 1), last + 1):
            page = order.pop()
            table[slots[b], a % ring] = page
            m = min(n, a * PAGE + PAGE) - a * PAGE
            kp[page, :, :m] = k[a * PAGE:a * PAGE + m].transpose(0, 1)
            vp[page, :, :, :m] = v[a * PAGE:a * PAGE + m].permute(1, 2, 0)
        d, s = random_tree(nodes[b], g, chain) if nodes[b] else ([], [])
        depths.append(d)
        seen.append(s)
    T = sum(nodes)
    words = words or max(1, (max(nodes) + 63) // 64)
    return dict(held=held, nodes=nodes, lens=lens, ring=ring, n_heads=n_heads, n_kv=n_kv, hd=hd, dtype=dtype, window=window, kp=kp, vp=vp, table=table,
                slots=slots, keys=keys, vals=vals, depths=depths, seen=seen, words=words, q=rnd((T, n_heads * hd), seed + 3, dtype))


def tree_rows(c):
    """For every row: (sequence, node, the positions that it sees)."""
    for b, (h, n) in enumerate(zip(c["held"], c["nodes"])):
        for i in range(n):
            lo = max(0, h + c["depths"][b][i] - c["window"] + 1) if c["window"] else 0
            yield b, i, list(range(lo, h)) + [h + j for j in range(n) if c["seen"][b][i] >> j & 1]


def tree_reference(c):
    """(result, what a result may be off by) float64 [T, heads, hd] each.  A rounding to storage type is half a step (2^-8 in bfloat16) of the
    result; in bfloat16 the probabilities are rounded too, which moves a weighted mean by 2^-8 of the greatest |value|; float32 sums
    of head_dim products and of the keys, and exponentials of scores so formed, are off by 2^-24 of their terms each."""
    nh, hd, G = c["n_heads"], c["hd"], c["n_heads"] // c["n_kv"]
    q = c["q"].double().view(-1, nh, hd)
    want, lim = torch.zeros_like(q), torch.zeros_like(q)
    half = 2.0 ** -8 if c["dtype"] == torch.bfloat16 else 2.0 ** -24
    for r, (b, i, at) in enumerate(tree_rows(c)):
        if not at:
            continue
        k, v = c["keys"][b][at].double(), c["vals"][b][at].double()
        for h in range(nh):
            kk, vv = k[:, h // G], v[:, h // G]
            s = kk @ q[r, h] / math.sqrt(hd)
            want[r, h] = torch.softmax(s, 0) @ vv
            size = (kk.abs() @ q[r, h].abs()).max() / math.sqrt(hd)
            f32 = (2 * (hd + 4) * size + len(at) + 64) * 2.0 ** -24 * vv.abs().max()
            lim[r, h] = half * (want[r, h].abs() + (vv.abs().max() if half > 1e-6 else 0)) + f32
    return want, lim


def run_tree(c, splits=None, positions=True, simple=False, spare=2, out=None, step_max_len=True):
    k = K()
    T = sum(c["nodes"])
    kp, vp = pages_as_stored(c["kp"], c["vp"])
    width = c["n_heads"] * c["hd"]
    q = torch.cat([c["q"], torch.full((spare, width), float("nan"), dtype=c["dtype"])]).to(DEV)
    if out is None:
        out = torch.full((T + spare, width), 77.0, dtype=c["dtype"], device=DEV)
    mask = torch.cat([words_of([m for s in c["seen"] for m in s], c["words"]).view(-1, c["words"]), torch.full((spare, c["words"]), -1)]).to(DEV)
    pos = i32([h + d for h, ds in zip(c["held"], c["depths"]) for d in ds] + [0] * spare) if positions else None
    cu = np.concatenate([[0], np.cumsum(c["nodes"])]).tolist()
    if splits is None:
        splits = k.attn_tree_splits(len(c["held"]), max(c["nodes"]), max(c["lens"]), c["n_heads"], c["n_kv"], c["hd"], c["dtype"], c["window"])
    partial = torch.full((k.attn_tree_workspace_floats(T + spare, c["n_heads"], c["hd"], splits),), float("nan"), device=DEV)
    k.FORCE_SIMPLE = simple
    try:
        k.attn_tree(q, kp.to(DEV), vp.to(DEV), c["table"].to(DEV), c["ring"], i32(c["slots"]), i32(c["lens"]), i32(cu), mask, out, partial, c["n_heads"],
                    c["n_kv"], c["hd"], c["window"], splits, max(c["nodes"]), positions=pos, step_max_len=i32([max(c["lens"])]) if step_max_len else None)
    finally:
        k.FORCE_SIMPLE = False
    assert (out[T:] == 77.0).all()                             # rows behind the last sequence
    return out[:T].cpu().double().view(T, c["n_heads"], c["hd"])


def check_tree(c, what="", **kw):
    want, lim = tree_reference(c)
    got = run_tree(c, **kw)
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - lim
    assert (off <= 0).all(), "%s: %.3e beyond what it may be off" % (what, off.max().item())


BOTH = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("simple", [False, True])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 128), (8, 1, 64), (3, 3, 16), (6, 2, 80), (2, 1, 6), (4, 4, 96), (2, 1, 160), (20, 1, 32), (5, 1, 112)])
def test_trees_of_every_head_size(heads, kv, hd, simple, dtype):
    check_tree(tree_case([70, 0, 9, 128], [5, 3, 17, 1], heads, kv, hd, dtype, seed=hd), "heads of %d" % hd, simple=simple)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("held,nodes", [([0], [1]), ([1], [1]), ([63], [1]), ([64], [1]), ([63], [2]), ([0], [64]), ([1], [64]), ([5], [65]), ([60], [130]),
                                        ([64], [256]), ([700], [33]), ([0, 500, 3, 64], [16, 1, 40, 7]), ([300] * 9, [12] * 9), ([129, 20], [0, 4])])
def test_trees_of_every_length(held, nodes, dtype):
    check_tree(tree_case(held, nodes, 8, 2, 64, dtype, seed=len(held) + nodes[0]), "%s %s" % (held, nodes))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("splits", [1, 2, 5, 16])
@pytest.mark.parametrize("step_max_len", [True, False])
def test_trees_cut_into_pieces(splits, step_max_len, dtype):
    c = tree_case([1000, 64, 0, 300], [21, 3, 9, 40], 8, 2, 128, dtype, seed=splits)
    check_tree(c, "%d splits" % splits, splits=splits, step_max_len=step_max_len)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("window", [1, 5, 64, 100, 257])
@pytest.mark.parametrize("positions", [True, False])
def test_trees_behind_a_window(window, positions, dtype):
    """Nodes deeper than the window's width see no held token; without positions a node's place follows from its ancestors."""
    c = tree_case([400, 3, 64, 130], [12, 9, 30, 1], 4, 2, 64, dtype, window=window, seed=window, chain=True)
    check_tree(c, "window %d" % window, positions=positions, splits=3)
    c = tree_case([200, 40], [20, 9], 4, 2, 128, dtype, window=window, seed=window)
    check_tree(c, "window %d" % window, positions=positions)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("simple", [False, True])
def test_rows_that_see_nothing_and_sequences_without_a_slot(simple, dtype):
    c = tree_case([0, 30, 80], [6, 4, 7], 4, 2, 64, dtype, seed=4)
    c["seen"][0] = [0, 0b11, 0, 0b101, 0b100000, 0]            # what a mask names need not be a tree
    c["seen"][2][3] = 0                                        # only the held tokens
    c["slots"][1] = -1
    want, lim = tree_reference(c)
    got = run_tree(c, simple=simple)
    for r in (0, 2, 5, 6, 7, 8, 9):
        assert (got[r] == 0).all(), r
    live = [1, 3, 4] + list(range(10, 17))
    assert ((got - want).abs() <= lim)[live].all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("simple", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(bad, simple, dtype):
    """A drafted token whose key and value are no numbers reaches the rows whose masks name it and no other one; so does a token
    behind the window."""
    c = tree_case([90], [12], 4, 2, 64, dtype, window=60, seed=6)
    node = 3
    where = [(90 + node, [r for r, (_, _, at) in enumerate(tree_rows(c)) if 90 + node in at]),
             (31, [r for r, (_, _, at) in enumerate(tree_rows(c)) if 31 in at])]
    assert all(0 < len(rows) < 12 for _, rows in where)
    for pos, rows in where:
        d = dict(c, kp=c["kp"].clone(), vp=c["vp"].clone())
        page = int(c["table"][c["slots"][0], pos // PAGE % c["ring"]])
        d["kp"][page, :, pos % PAGE] = bad
        d["vp"][page, 1, 5:9, pos % PAGE] = bad
        got = run_tree(d, simple=simple)
        want, lim = tree_reference(c)
        free = [r for r in range(12) if r not in rows]
        assert torch.isfinite(got[free]).all() and ((got - want).abs() <= lim)[free].all()
        assert not torch.isfinite(got[rows]).all(dim=-1)[:, 2:].any()           # the heads of the KV head whose value it is
        e = dict(c, kp=c["kp"], vp=c["vp"].clone())            # the value alone
        e["vp"][page, 1, 5:9, pos % PAGE] = bad
        got = run_tree(e, simple=simple)
        assert torch.isfinite(got[free]).all() and ((got - want).abs() <= lim)[free].all()
        odd = got[rows][:, 2:, 5:9]
        assert (torch.isnan(odd) if bad != bad else odd == bad).all()
        rest = got[rows].clone()
        rest[:, 2:, 5:9] = want[rows][:, 2:, 5:9]
        assert ((rest - want[rows]).abs() <= lim[rows]).all()


def test_trees_far_into_a_long_cache():
    """Pages whose elements lie beyond 2^31 from the pool's start: 16,400 pages of 16 heads of 128 are 2.1 billion elements."""
    n_pages, H, hd = 16400, 16, 128
    kp = torch.zeros((n_pages, H, PAGE, hd), dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros((n_pages, H, hd, PAGE), dtype=torch.bfloat16, device=DEV)
    c = tree_case([130], [9], 16, 16, hd, torch.bfloat16, seed=8)
    ks, vs = pages_as_stored(c["kp"], c["vp"])
    far = [n_pages - 1 - i for i in range(c["ring"])]
    for col, page in enumerate(far):
        kp[page], vp[page] = ks[int(c["table"][c["slots"][0], col])].to(DEV), vs[int(c["table"][c["slots"][0], col])].to(DEV)
    table = torch.full((3, c["ring"]), -1, dtype=torch.int32)
    table[1] = torch.tensor(far)
    out = torch.empty((9, 16 * hd), dtype=torch.bfloat16, device=DEV)
    splits = K().attn_tree_splits(1, 9, 139, 16, 16, hd, torch.bfloat16)
    partial = torch.empty(K().attn_tree_workspace_floats(9, 16, hd, splits), device=DEV)
    mask = words_of(c["seen"][0], 1).to(DEV)
    K().attn_tree(c["q"].to(DEV), kp, vp, table.to(DEV), c["ring"], i32([1]), i32([139]), i32([0, 9]), mask, out, partial, 16, 16, hd, 0, splits, 9)
    want, lim = tree_reference(c)
    assert ((out.cpu().double().view(9, 16, hd) - want).abs() <= lim).all()
    # copies and moves there, too
    K().copy_pages(kp[None], vp[None], i32([far[0]]), i32([n_pages - 100]))
    assert torch.equal(kp[n_pages - 100], kp[far[0]]) and torch.equal(vp[n_pages - 100], vp[far[0]])
    K().compact_lines(kp[None], vp[None], table.to(DEV), c["ring"], i32([1]), i32([130]), i32([0, 2]), i32([0, 5]), 2)
    kr, vr = pages_as_rows(kp[far[2]][None].cpu(), vp[far[2]][None].cpu())
    assert torch.equal(kr[0, :, 3], c["keys"][0][135]) and torch.equal(vr[0, :, :, 3], c["vals"][0][135])


@pytest.mark.parametrize("dtype", BOTH)
def test_trees_in_a_graph_and_the_same_bits_twice(dtype):
    c = tree_case([500, 77], [20, 33], 8, 2, 128, dtype, seed=12)
    k = K()
    kp, vp = (x.to(DEV) for x in pages_as_stored(c["kp"], c["vp"]))
    q, mask = c["q"].to(DEV), words_of([m for s in c["seen"] for m in s], 1).to(DEV)
    table, slots, lens, cu = c["table"].to(DEV), i32(c["slots"]), i32(c["lens"]), i32([0, 20, 53])
    out = torch.zeros_like(q)
    partial = torch.empty(k.attn_tree_workspace_floats(53, 8, 128, 4), device=DEV)

    def go():
        k.attn_tree(q, kp, vp, table, c["ring"], slots, lens, cu, mask, out, partial, 8, 2, 128, 0, 4, 33)

    go()
    first = out.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for i in range(3):
        out.zero_()
        partial.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
        go()
        assert torch.equal(out, first)
    want, lim = tree_reference(c)
    assert ((first.cpu().double().view(53, 8, 128) - want).abs() <= lim).all()


# ------------------------------------------------------------------------------------------------ trees over LDS, by how many columns a workgroup takes
def columns_of(c):
    """How many columns (nodes times the heads of a group) a workgroup of the bfloat16 kernels takes."""
    cols = max(c["nodes"]) * (c["n_heads"] // c["n_kv"])
    if cols <= 32 or c["hd"] % 32:
        return 16 if cols <= 16 else 32
    if cols <= 64:
        return 64
    units = torch.cuda.get_device_properties(0).multi_processor_count
    return 256 if cols > 128 and 2 * len(c["nodes"]) * c["n_kv"] > units else 128


@pytest.mark.parametrize("hd", [128, 32])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("splits", [None, 3])
def test_trees_with_all_columns_in_one_workgroup(hd, window, splits):
    """Sequences enough that more than 128 columns go in one workgroup: in one launch sequences that all eight waves share by columns, ones
    that two groups of waves share by pages, ones of a single tile and ones without nodes; contexts from none to several pages."""
    nodes = [61, 1, 33, 45, 0, 16, 61, 32, 5, 40, 48, 2, 61, 17, 34, 9, 58, 3, 37, 61, 20, 33, 64, 31]
    held = [0, 1, 63, 64, 65, 127, 200, 300, 5, 129, 191, 400, 64, 2, 250, 33, 128, 90, 61, 3, 0, 150, 448, 320]
    c = tree_case(held, nodes, 32, 8, hd, torch.bfloat16, window=window, seed=hd + window)
    assert columns_of(c) == 256 and len(nodes) == len(held) == 24
    check_tree(c, "hd %d window %d splits %s" % (hd, window, splits), splits=splits)


FORMS = {64: (1, 4, 1, 12), 128: (2, 8, 2, 30), 1280: (2, 8, 2, 50), 256: (17, 32, 8, 45)}       # columns -> sequences, heads, KV heads, nodes; 1280: two workgroups of 128


@pytest.fixture(scope="module")
def lds_cases():
    """Each form's case and what it gives, worked out once."""
    made = {}

    def get(form, hd):
        if (form, hd) not in made:
            B, heads, kv, nodes = FORMS[form]
            held = [150] + [10 + 7 * b for b in range(1, B)]
            c = tree_case(held, [nodes] * B, heads, kv, hd, torch.bfloat16, window=130, seed=form + hd)
            assert columns_of(c) == {1280: 128}.get(form, form)
            made[form, hd] = (c,) + tree_reference(c)
        return made[form, hd]

    return get


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("splits", [1, 2])
def test_what_a_row_does_not_see_does_not_reach_it_over_lds(lds_cases, splits, bad, form, hd):
    """As for few columns: a drafted token, one at the window's edge and one that every row sees, whose values (and keys) are no numbers,
    on both of a round's pages: they reach the rows that see them and no other, and leave every other element as it is."""
    c, want, lim = lds_cases(form, hd)
    B, heads, kv, nodes = FORMS[form]
    G = heads // kv
    rows_of = list(tree_rows(c))
    elements = [5, 6, 7, 8, hd - 1]
    for pos in (150 + 3, 150 + nodes - 1, 22, 100):
        rows = [r for r, (b, _, at) in enumerate(rows_of) if b == 0 and pos in at]
        assert 0 < len(rows) and (pos != 100 or len(rows) == nodes)
        free = sorted(set(range(len(rows_of))) - set(rows))
        page = int(c["table"][c["slots"][0], pos // PAGE % c["ring"]])
        g = kv - 1
        e = dict(c, vp=c["vp"].clone())                        # the value alone
        e["vp"][page, g, elements, pos % PAGE] = bad
        got = run_tree(e, splits=splits)
        assert torch.isfinite(got[free]).all() and ((got - want).abs() <= lim)[free].all(), (pos, "rows that do not see it")
        odd = got[rows][:, g * G:][..., elements]
        assert (torch.isnan(odd) if bad != bad else odd == bad).all(), (pos, "rows that see it")
        rest = got[rows].clone()
        for x in elements:
            rest[:, g * G:, x] = want[rows][:, g * G:, x]
        assert ((rest - want[rows]).abs() <= lim[rows]).all(), (pos, "the other elements")
        d = dict(e, kp=c["kp"].clone())                        # the key too
        d["kp"][page, g, pos % PAGE] = bad
        got = run_tree(d, splits=splits)
        assert torch.isfinite(got[free]).all() and ((got - want).abs() <= lim)[free].all(), (pos, "keys")
        assert not torch.isfinite(got[rows][:, g * G:]).all(dim=-1).any()


def test_the_splits_count_this_card_s_units():
    """attn_tree_splits has the compute units written out that the kernels' own choice of columns asks the card for."""
    assert torch.cuda.get_device_properties(0).multi_processor_count == 256
    for B in (16, 17):                                         # 2 x 16 x 8 halves all run at once, 2 x 17 x 8 do not
        c = dict(nodes=[61] * B, n_heads=32, n_kv=8, hd=128)
        chunks = -(-61 * 4 // columns_of(c))
        assert K().attn_tree_splits(B, 61, 100000, 32, 8, 128, torch.bfloat16) == max(1, 256 // (B * 8 * chunks))
