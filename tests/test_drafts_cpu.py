"""Refusals of the operators around drafted tokens, without a GPU: every check of arguments stands in front of the launch."""
import pytest
import torch

from yalm_amd.ops import kernels


def test_tensors_that_are_not_on_the_gpu_are_refused():
    x = torch.zeros((2, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.sample_filtered(x, torch.zeros(2), torch.zeros(2, dtype=torch.int32))
    pages = torch.zeros((1, 2, 1, 64, 16)), torch.zeros((1, 2, 1, 16, 64))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.copy_pages(*pages, i, i)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.compact_lines(*pages, torch.zeros((1, 1), dtype=torch.int32), 1, i, i, torch.zeros(2, dtype=torch.int32), i, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.attn_tree(torch.zeros((1, 16)), pages[0][0], pages[1][0], torch.zeros((1, 1), dtype=torch.int32), 1, i, i, torch.zeros(2, dtype=torch.int32),
                          torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 16)), torch.zeros(0), 1, 1, 16, 0, 1, 1)


def test_tensors_of_another_device_are_refused(monkeypatch):
    class OnSecond(torch.Tensor):                      # a tensor that says it lies on the second GPU
        is_cuda = True

        def get_device(self):
            return 1

    def on_second(*a, **kw):
        return torch.zeros(*a, **kw).as_subclass(OnSecond)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    i, cu, i2 = on_second(1, dtype=torch.int32), on_second(2, dtype=torch.int32), on_second((1, 1), dtype=torch.int32)
    k, v = on_second((1, 2, 1, 64, 16)), on_second((1, 2, 1, 16, 64))
    with pytest.raises(RuntimeError, match="device 1"):
        kernels.sample_filtered(on_second((2, 8)), on_second(2), cu)
    with pytest.raises(RuntimeError, match="device 1"):
        kernels.copy_pages(k, v, i, i)
    with pytest.raises(RuntimeError, match="device 1"):
        kernels.compact_lines(k, v, i2, 1, i, i, cu, i, 1)
    with pytest.raises(RuntimeError, match="device 1"):
        kernels.attn_tree(on_second((1, 16)), k[0], v[0], i2, 1, i, i, cu, on_second((1, 1), dtype=torch.int64), on_second((1, 16)), on_second(0), 1, 1, 16, 0,
                          1, 1)


def test_the_command_line_s_settings_are_checked():
    from yalm_amd import cli
    for bad in (["--draft", "256"], ["--draft", "-1"], ["--top-p", "1.5"], ["--min-p", "-1"], ["--top-k", "-2"], ["--samples", "0"], ["--draft", "2", "--samples", "2"]):
        with pytest.raises(SystemExit):
            cli.parse_args(["folder", "-i", "text"] + bad)
    assert cli.parse_args(["folder", "-i", "text", "--draft", "255"])["draft"] == 255


def test_shapes_that_say_nothing_are_refused():
    with pytest.raises(ValueError, match="vocabulary"):
        kernels.sample_filtered(torch.zeros(8), None, None)
    with pytest.raises(ValueError, match="vocabulary"):
        kernels.sample_filtered(torch.zeros((2, 0)), None, None)
    with pytest.raises(ValueError, match="lines, pages"):
        kernels.compact_lines(torch.zeros((2, 64, 16)), None, None, 1, None, None, None, None, 1)
    with pytest.raises(ValueError, match="multiple"):
        kernels.attn_tree(None, None, None, None, 1, None, None, None, None, None, None, 3, 2, 64, 0, 1, 1)


@pytest.mark.parametrize("wrong", [dict(n_heads=3), dict(head_dim=0), dict(head_dim=2048), dict(ring=0), dict(ring=9), dict(n_slots=0), dict(words=0), dict(n_splits=0),
                                   dict(max_nodes=0), dict(max_nodes=257), dict(n_pages=0), dict(layout=1, head_dim=48), dict(dtype=7), dict(n_heads=65536, n_kv=1)])
def test_the_library_s_entry_refuses_numbers_that_name_no_step(wrong):
    """The C entry by itself, without memory behind its pointers: it answers before it would launch."""
    from yalm_amd.ops import library
    s = {**dict(T=5, B=1, n_heads=4, n_kv=2, head_dim=64, n_splits=1, max_nodes=5, n_pages=3, layout=1, dtype=0, ring=2, stride=8, n_slots=2, words=1), **wrong}
    code = library.lib().yalm_attn_tree(None, None, None, None, s["stride"], s["n_slots"], s["ring"], None, None, None, None, s["words"], None, None, None, s["T"], s["B"],
                                        s["n_heads"], s["n_kv"], s["head_dim"], 0, s["n_splits"], s["max_nodes"], s["n_pages"], s["layout"], s["dtype"], 0, None,
                                        None)
    assert code != 0
    with pytest.raises(Exception):
        library.check(code, "attn_tree")


def test_the_library_s_other_entries_refuse_too():
    from yalm_amd.ops import library
    lib = library.lib()
    assert lib.yalm_sample_filtered(None, None, None, None, None, None, None, None, None, 2, 0, None) != 0
    assert lib.yalm_sample_filtered(None, None, None, None, None, None, None, None, 8, 2, 100, None) != 0       # a workspace off 16 bytes
    assert lib.yalm_sample_filtered(None, None, None, None, None, None, None, None, None, 0, 100, None) == 0    # no rows
    assert lib.yalm_copy_blocks(None, None, 2, 3, 64, None, None, 1, None) != 0
    assert lib.yalm_copy_blocks(None, None, 2, 3, 64, None, None, 0, None) == 0
    for kw in (dict(ring=0), dict(ring=5), dict(slots=0), dict(lines=65536), dict(pages=0), dict(layout=1, hd=48), dict(B=65536)):
        s = {**dict(ring=2, slots=2, lines=2, pages=3, layout=1, hd=64, B=1), **kw}
        assert lib.yalm_compact_lines(None, None, None, 4, s["slots"], s["ring"], None, None, None, None, s["B"], 1, 1, s["lines"], s["pages"], 1, s["hd"], s["layout"], 0,
                                      None) != 0, kw


def test_workspace_sizes():
    assert kernels.attn_tree_workspace_floats(7, 4, 64, 1) == 0
    assert kernels.attn_tree_workspace_floats(7, 4, 64, 3) == 7 * 4 * 3 * 66
    assert kernels.sample_filtered_workspace(3, 32000) >= 0


# ------------------------------------------------------------------------------------------------ pages that are shared
def _cache(max_tokens=1024, window=0, n_slots=8, sinks=0, max_draft=0):
    from yalm_amd.cache import CacheManager, KVRequest, StateRequest
    req = {0: KVRequest(1, 4, window, sinks), 1: KVRequest(1, 4, window, sinks), 2: StateRequest((3,))}
    return CacheManager(req, max_tokens, max_tokens, torch.float32, "cpu", n_slots=n_slots, max_draft=max_draft)


def test_a_page_is_free_when_the_last_holder_gives_it_back():
    from yalm_amd.cache import CacheError, PagePool
    p = PagePool(2)
    a = p.take()
    p.share(a)
    assert p.holders(a) == 2 and p.n_free == 1
    p.give_back(a)
    assert p.holders(a) == 1 and p.n_free == 1
    p.give_back(a)
    assert p.n_free == 2
    for bad in (p.give_back, p.share):
        with pytest.raises(CacheError):
            bad(a)


def test_forks_share_full_pages_and_copy_the_last_one():
    c = _cache()
    (s,) = c.acquire(1)
    c.extend([s], [150])
    g = c.kv_groups[0]
    new, copies = c.fork(s, 2)
    table = g.table_host
    for t in new:
        assert c.seq_len[t] == 150 and (table[t, :2] == table[s, :2]).all() and table[t, 2] != table[s, 2]
    assert table[new[0], 2] != table[new[1], 2] and g.pool.holders(int(table[s, 0])) == 3 and g.pool.n_free == 16 - 5
    (k, v, src, dst), (state, none, src_s, dst_s) = copies
    assert k is g.k_pages and v is g.v_pages and src == [int(table[s, 2])] * 2 and dst == [int(table[t, 2]) for t in new]
    assert state is c.state_groups[0].data and none is None and src_s == [s, s] and dst_s == new
    assert torch.equal(g.table, torch.from_numpy(table))
    c.extend([s] + new, [64, 1, 43])                   # each goes on in pages of its own
    assert len({int(table[t, 2]) for t in [s] + new}) == 3 and int(table[s, 3]) != int(table[new[1], 3]) >= 0
    c.release([s])
    assert g.pool.holders(int(table[new[0], 0])) == 2
    c.release(new)
    assert g.pool.n_free == g.n_pages and c.slots.n_free == 8
    (t,) = c.acquire(1)
    c.extend([t], [128])                               # a prompt that ends with its page: nothing to copy but the state
    new, copies = c.fork(t, 1)
    assert len(copies) == 1 and g.pool.n_free == 16 - 2


def test_forks_of_windows_and_sinks_are_copies_and_what_does_not_fit_changes_nothing():
    from yalm_amd.cache import CacheError, CacheFull
    c = _cache(window=100, sinks=2)
    (s,) = c.acquire(1)
    c.extend([s], [500])
    g = c.kv_groups[0]
    new, copies = c.fork(s, 1)
    assert g.ring_pages == 3 and len(copies) == 3 and copies[0][2] == [int(p) for p in g.table_host[s]] and copies[1][0] is g.sink_k
    assert g.pool.n_free == 16 - 6
    free = (g.pool.n_free, c.slots.n_free, g.table_host.copy())
    with pytest.raises(CacheFull, match="pages"):
        c.fork(s, 4)
    with pytest.raises(CacheFull, match="slots"):
        c.fork(s, 9)
    for bad in ((7, 1), (s, -1)):
        with pytest.raises(CacheError):
            c.fork(*bad)
    assert (g.pool.n_free, c.slots.n_free) == free[:2] and (g.table_host == free[2]).all()
    assert c.fork(s, 0) == ([], [])


@pytest.mark.parametrize("window", [0, 100])
def test_cut_sequences_give_back_their_pages(window):
    from yalm_amd.cache import CacheError
    c = _cache(window=window, max_draft=70)
    g = c.kv_groups[0]
    assert g.ring_pages == (16 if not window else (100 + 69 + 63) // 64 + 1)
    (s,) = c.acquire(1)
    for base, more, to in ((60, 70, 61), (61, 3, 64), (64, 64, 64), (64, 65, 65), (65, 63, 128), (300, 70, 310)):
        c.extend([s], [base - c.seq_len[s]] if base > c.seq_len[s] else [0]) if base != c.seq_len[s] else None
        c.extend([s], [more])
        c.cut([s], [to])
        held = [int(p) for p in g.table_host[s] if p >= 0]
        assert c.seq_len[s] == to and len(held) == len(set(held)) and g.pool.n_free == 16 - len(held)
        assert len(held) == min((to + 63) // 64, g.ring_pages) or window
    for bad in (-1, 311):
        with pytest.raises(CacheError):
            c.cut([s], [bad])
    c.release([s])
    assert g.pool.n_free == 16


# ------------------------------------------------------------------------------------------------ guesses
def test_guesses_from_a_text_itself():
    from yalm_amd.drafting import _shallow, accept, lookup_tree
    text = [5, 6, 7, 8, 9, 1, 5, 6, 7, 2, 3, 5, 6]
    tokens, parents = lookup_tree(text, 7)
    assert tokens == [6, 7, 2, 3, 8, 9] and parents == [-1, 0, 1, 2, 1, 4]        # the later place first, the common 7 once
    assert lookup_tree([4], 5) == ([4], [-1]) and lookup_tree([1, 2, 3], 5) == ([3], [-1])
    assert lookup_tree(text, 1) == ([6], [-1])
    for n in range(1, 30):
        tokens, parents = lookup_tree([1, 2] * 20, n)
        assert len(tokens) <= n and parents[0] == -1 and all(p < j for j, p in enumerate(parents))
    tokens, parents = [6, 7, 2, 3, 8, 9], [-1, 0, 1, 2, 1, 4]
    assert accept(tokens, parents, [7, 8, 0, 0, 9, 4]) == ([0, 1, 4, 5], [7, 8, 9, 4])
    assert accept(tokens, parents, [1, 8, 0, 0, 9, 4]) == ([0], [1])
    assert accept(tokens, parents, [7, 2, 3, 6, 0, 0]) == ([0, 1, 2, 3], [7, 2, 3, 6])
    assert _shallow(tokens, parents, 2) == ([6, 7], [-1, 0], [0, 1])
    assert _shallow(tokens, parents, 3) == ([6, 7, 2, 8], [-1, 0, 1, 1], [0, 1, 2, 2])
    assert _shallow(tokens, parents, 1) == ([6], [-1], [0])


def test_command_line_settings():
    from yalm_amd.cli import parse_args
    a = parse_args(["folder", "--tokens", "1,2", "--top-k", "40", "--top-p", "0.9", "--min-p", "0.05", "--samples", "3"])
    assert (a["top_k"], a["top_p"], a["min_p"], a["samples"], a["draft"]) == (40, 0.9, 0.05, 3, 0)
    assert parse_args(["folder", "--tokens", "1,2", "--draft", "8"])["draft"] == 8
    d = parse_args(["folder", "--tokens", "1,2"])
    assert (d["top_k"], d["top_p"], d["min_p"], d["samples"], d["draft"]) == (0, 1.0, 0.0, 1, 0)
    for bad in (["--top-k", "-1"], ["--top-p", "1.2"], ["--min-p", "-0.1"], ["--samples", "0"], ["--draft", "-2"], ["--draft", "2", "--samples", "2"]):
        with pytest.raises(SystemExit):
            parse_args(["folder", "--tokens", "1,2"] + bad)


# ------------------------------------------------------------------------------------------------ rings and what their windows see
def _windows(max_tokens, max_seq_len, windows=(100,), n_slots=4, **kw):
    from yalm_amd.cache import CacheManager, KVRequest
    return CacheManager({i: KVRequest(1, 4, w) for i, w in enumerate(windows)}, max_tokens, max_seq_len, torch.float32, "cpu", n_slots=n_slots, **kw)


class Lines:
    """What a ring's pages hold, written as the kernels write them: whole prompts by pages, later tokens one place each."""

    def __init__(self, c):
        self.c, self.at = c, {}

    def grow(self, slot, n):
        old = self.c.seq_len[slot]
        (new,) = self.c.extend([slot], [n])
        for i, g in enumerate(self.c.kv_groups):
            for pos in range(old, new):
                if old > 0 or pos // 64 > (new - 1) // 64 - g.ring_pages:
                    page = int(g.table_host[slot, pos // 64 % g.ring_pages])
                    assert 0 <= page < g.n_pages
                    self.at[i, page, pos % 64] = (slot, pos)
        return old, new

    def check(self, slot, old, new):
        """Every key that the tokens at old ... new - 1 see is held, the drafted ones themselves too."""
        for i, g in enumerate(self.c.kv_groups):
            for pos in range(max(0, old - g.window + 1), new):
                assert self.at[i, int(g.table_host[slot, pos // 64 % g.ring_pages]), pos % 64] == (slot, pos), (i, pos, old, new)


@pytest.mark.parametrize("windows,max_tokens,max_seq_len,max_draft,refuses",
                         [((4096,), 256, 8192, 32, True), ((1024,), 4096, 1024, 8, False), ((1024,), 1024, 1024, 8, True), ((100,), 128, 400, 70, True),
                          ((100, 300), 256, 1000, 9, True), ((62,), 64, 4000, 0, True), ((100,), 1024, 1024, 70, False), ((64,), 320, 64, 17, False)])
def test_drafted_tokens_never_lie_on_keys_that_a_window_sees(windows, max_tokens, max_seq_len, max_draft, refuses):
    """Prompts and trees of any size: what is not refused keeps all that it sees, and a refusal changes nothing."""
    from yalm_amd.cache import CacheFull
    rng = __import__("random").Random(max_tokens + max_draft)
    went_on = refused = 0
    for prompt in (1, 30, 63, 64, 65, 90, 150, 250, 1010):
        c = _windows(max_tokens, max_seq_len, windows, max_draft=max_draft)
        lines = Lines(c)
        (s,) = c.acquire(1)
        if prompt > max_seq_len:
            continue
        lines.grow(s, prompt)
        for _ in range(300):
            n = rng.randint(1, max(1, max_draft)) if rng.random() < 0.5 else 1
            before = (c.seq_len[s], [g.pool.n_free for g in c.kv_groups], [g.table_host.copy() for g in c.kv_groups], c.room(s))
            if before[0] + n > max_seq_len + max_draft:
                break
            try:
                lines.check(s, *lines.grow(s, n))
                went_on += 1
                assert n <= before[3]
            except CacheFull:
                refused += 1
                assert before[:2] == (c.seq_len[s], [g.pool.n_free for g in c.kv_groups]) and all((a == g.table_host).all() for a, g in zip(before[2], c.kv_groups))
                assert n > before[3]
                if before[3] < 1:
                    break
                continue
            c.cut([s], [before[0] + rng.randint(1, n)])
        c.release([s])
        assert all(g.pool.n_free == g.n_pages for g in c.kv_groups)
    assert went_on > 40 and (refused > 0) == refuses


def test_rings_have_room_for_drafts_up_to_the_end_of_the_context():
    c = _windows(4096, 1024, (1024,), max_draft=8)
    assert c.kv_groups[0].ring_pages == 17
    (s,) = c.acquire(1)
    c.extend([s], [1019])
    assert c.extend([s], [8]) == [1027] and c.kv_groups[0].pool.n_free == 64 - 17
    assert _windows(4096, 1024, (1024,)).kv_groups[0].ring_pages == 16           # without drafts no sequence is longer
    assert _windows(4096, 64, (62,), longest=500).kv_groups[0].ring_pages == 2   # a text that runs past the model's positions
    assert _windows(64, 64, (62,), longest=500).kv_groups[0].ring_pages == 1


def test_a_sequence_that_outgrows_a_small_cache_is_refused():
    """The window is wider than all pages together: the prompt itself may be longer (its own keys are staged), but nothing goes on where a
    key in sight is gone."""
    from yalm_amd.cache import CacheFull
    c = _windows(256, 8192, (4096,))
    a, b = c.acquire(2)
    c.extend([a], [256])
    with pytest.raises(CacheFull, match="window"):
        c.extend([a], [1])
    assert c.seq_len[a] == 256 and c.room(a) == 0
    c.release([a])
    c.extend([b], [300])
    with pytest.raises(CacheFull, match="window"):
        c.extend([b], [1])
    c.release([b])
    (a,) = c.acquire(1)                                # nothing of the last sequence sticks to its slot
    c.extend([a], [100])
    assert c.extend([a], [150]) == [250] and c.room(a) == 6


def test_forks_of_short_rings_know_what_is_gone():
    from yalm_amd.cache import CacheFull
    c = _windows(256, 8192, (100,), max_draft=70)
    assert c.kv_groups[0].ring_pages == 4
    c = _windows(128, 8192, (100,), max_draft=70)
    (a,) = c.acquire(1)
    c.extend([a], [10])
    (b,), _ = c.fork(a, 1)
    assert c.room(b) == c.room(a) == 118
    c.release([a, b])
    (a,) = c.acquire(1)
    c.extend([a], [129])                               # pages 1 and 2 are held, position 129 sees from 30 on
    with pytest.raises(CacheFull, match="window"):
        c.extend([a], [1])


def test_cuts_that_would_write_on_for_others_are_refused():
    """A page that a fork shares is whole for everyone who holds it: who were cut into one would write on in it."""
    from yalm_amd.cache import CacheError
    c = _windows(1024, 1024, (0, 100))
    a, z = c.acquire(2)
    c.extend([a, z], [150, 10])
    (b,), _ = c.fork(a, 1)
    g = c.kv_groups[0] if c.kv_groups[0].window == 0 else c.kv_groups[1]

    def state():
        return list(c.seq_len), [(h.pool.n_free, h.table_host.tolist()) for h in c.kv_groups]

    before = state()
    for slots, lengths in (([a], [127]), ([b], [100]), ([b], [1]), ([z, a], [5, 70]), ([a, a], [149, 150]), ([a, a], [150, 149]), ([a, z], [150]), ([z], [11])):
        with pytest.raises(CacheError):
            c.cut(slots, lengths)
        assert state() == before
    c.cut([a, b], [130, 128])                          # behind what they share
    assert g.pool.holders(int(g.table_host[a, 0])) == 2 and (g.table_host[b, 2:] == -1).all()
    c.extend([b], [3])
    assert int(g.table_host[b, 2]) != int(g.table_host[a, 2])
    c.cut([b], [64])                                   # a page's end: the next token starts a page of its own
    c.extend([b], [1])
    assert int(g.table_host[b, 0]) == int(g.table_host[a, 0]) and g.pool.holders(int(g.table_host[b, 1])) == 1 and g.table_host[b, 1] != g.table_host[a, 1]
    c.release([b])
    c.cut([a], [100])                                  # nobody else holds it any more
    c.release([a, z])
    assert all(h.pool.n_free == h.n_pages for h in c.kv_groups)


@pytest.mark.parametrize("max_tokens", [1024, 128])
def test_cuts_to_where_a_window_s_keys_are_gone_are_refused(max_tokens):
    from yalm_amd.cache import CacheError
    c = _windows(max_tokens, 8192, (100,), max_draft=20)
    lines = Lines(c)
    (a,) = c.acquire(1)
    lines.grow(a, 90)
    for _ in range(300):
        lines.grow(a, 1)
    ring = c.kv_groups[0].ring_pages * 64
    assert ring == (192 if max_tokens == 1024 else 128)
    first, more = 390 - ring + 99, 63 if max_tokens == 1024 else 20      # from `first` on the next token sees what is held; pages count whole
    with pytest.raises(CacheError, match="window"):
        c.cut([a], [first - 64])
    assert c.seq_len[a] == 390
    c.cut([a], [first + more])
    lines.check(a, *lines.grow(a, 1))
    c.cut([a], [first + more])
    with pytest.raises(CacheError, match="window"):    # what was written behind does not come back by steps
        for n in range(first + more - 1, first - 65, -1):
            c.cut([a], [n])
            old, new = lines.grow(a, 1)
            lines.check(a, old, new)


# ------------------------------------------------------------------------------------------------ the drafting loop without a GPU
class ScriptedDrafts:
    """An engine whose model says at each place of request r the token 7 r + place: nothing but the loop's decisions is run."""
    max_draft, max_draft_depth = 256, 256

    class _Cache:
        unbounded, max_seq_len = False, 4096

        def __init__(self, n_slots, n_pages):
            self.n_slots, self.n_pages = n_slots, n_pages

        def room(self, slot):
            return 1 << 30

        def whole_rings(self):
            return 0

    def __init__(self, n_slots=8, n_pages=400, n_positions=4096, most=None):
        self.cache, self.n_positions = self._Cache(n_slots, n_pages), n_positions
        self.lens, self.sizes, self.free, self.pending = {}, [], list(range(n_slots)), {}
        if most is not None:
            self.max_step_drafts = most

    def start(self, n):
        out = [self.free.pop(0) for _ in range(n)]
        self.lens.update({s: 0 for s in out})
        return out

    def release(self, slots):
        for s in slots:
            del self.lens[s]
            self.free.append(s)

    def length(self, slot):
        return self.lens[slot]

    def step_bytes(self, slots):
        return 0

    def step(self, slots, tokens):
        for s, t in zip(slots, tokens):
            self.lens[s] += len(t)
        return None

    def draft_step(self, slots, tokens, parents):
        assert all(len(p) == len(t) for p, t in zip(parents, tokens))
        self.sizes.append([len(t) for t in tokens])
        assert sum(self.sizes[-1]) <= getattr(self, "max_step_drafts", 1 << 30)
        return None

    def keep(self, slots, paths):
        for s, path in zip(slots, paths):
            self.lens[s] += len(path)


class ScriptedTokens:
    def sample(self, logits, temperature, request_ids, steps):
        return [7 * r + s for r, s in zip(request_ids, steps)]


def chain_guess(history, n):
    return [history[-1] + k for k in range(n)], list(range(-1, n - 1))


@pytest.mark.parametrize("most", [None, 1000, 100, 17, 8])
def test_a_step_s_drafts_stay_within_the_engine_s_limit(most):
    """Trees of a full batch are cut to what one step takes, in place of a refusal behind the prompts, with all results lost."""
    from yalm_amd import generate_drafted
    engine = ScriptedDrafts(most=1 << 30 if most is None else most)
    out = generate_drafted(engine, [[5] * (i + 1) for i in range(8)], max_new_tokens=300, stop_ids=[], sampler=ScriptedTokens(), guess=chain_guess, max_nodes=64)
    assert out == [[7 * r + s for s in range(300)] for r in range(8)]
    assert max(max(x) for x in engine.sizes) == min(64, (most or 1 << 30) // 8 if most != 17 else 2) and not engine.lens


# ------------------------------------------------------------------------------------------------ models without drafts
def _design(module):
    return next(v for k, v in vars(module).items() if k.isupper() and isinstance(v, dict) and "layers" in v)


def test_models_say_why_they_take_no_drafts():
    """The reason is the layer's own: state, sinks, a term by the distance, or an arrangement around plain attention that offers none."""
    import bovozen_configs
    import gedunex_configs
    import gemepel_configs
    import situlorn_configs
    import tiny_configs
    import zebivik_configs
    from yalm_amd import Model, config_from_dict
    plain = config_from_dict(tiny_configs.ALL["tiny_llama"])
    assert Model(plain.to_spec()).draft_refusal() == "" and Model(plain.to_spec()).takes_drafts()
    sinks = Model(plain.with_context(20).to_spec())
    assert not sinks.takes_drafts() and "layer 0" in sinks.draft_refusal() and "sinks" in sinks.draft_refusal()
    said = {}
    for module in (bovozen_configs, gedunex_configs, gemepel_configs, situlorn_configs, zebivik_configs):
        model = Model(config_from_dict(_design(module)).to_spec())
        said[module.__name__] = model.draft_refusal()
        assert not model.takes_drafts() and said[module.__name__]
    for name, why in (("gedunex", "ParallelResidualBlock"), ("gemepel", "embedding"), ("situlorn", "PostNormResidualBlock"), ("zebivik", "SandwichResidualBlock"),
                      ("bovozen", "mixer")):
        assert why in said[name + "_configs"], said
