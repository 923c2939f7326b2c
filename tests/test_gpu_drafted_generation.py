"""Drafted tokens, forked sequences and filtered sampling through the engine and the generation loops: a tree's logits against
the plain implementation on each node's own text, what is kept of it against the text without drafts, and the loops' tokens against the
ones that generate() gives without them."""
import numpy as np
import pytest
import torch

import bovozen_configs
import gemepel_configs
import helpers
import tiny_configs
import zebivik_configs
from plain import reference_model as R
from test_gpu_drafts import sample_reference

pytestmark = pytest.mark.gpu
NAMES = ["tiny_llama", "tiny_mistral", "tiny_llama3", "tiny_wide_heads"]


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("draft_models")
    return {name: helpers.make_folder(tmp, name, tiny_configs.ALL[name], seed=8) for name in NAMES}


def engine_of(folders, name, dtype, **kw):
    from yalm_amd import Engine, Model
    return Engine(Model.from_folder(folders[name], dtype=dtype, device="cuda:0"), **{"max_tokens": 1024, "max_batch": 6, "max_draft": 20, **kw})


def tree(n, seed):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(0, j - 4), j)) for j in range(1, n)]


def path_to(parents, j):
    out = []
    while j >= 0:
        out.append(j)
        j = parents[j]
    return out[::-1]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", NAMES)
def test_a_tree_s_logits_and_what_is_kept_of_it(folders, name, dtype):
    """Trees of several sizes behind prompts of several lengths (past the window of the Mistral one, over a page's end), three rounds of
    them, a plain step behind each: every logit is that of the node's own text."""
    engine = engine_of(folders, name, helpers.torch_dtype(dtype))
    cfg = tiny_configs.ALL[name]
    V, limit = cfg["vocab_size"], engine.n_positions
    rng = np.random.default_rng(3)
    texts = [rng.integers(0, V, n).tolist() for n in (1, 17, min(limit - 30, 59))]
    slots = engine.start(3)
    engine.step(slots, texts)

    def check(got, text, what):
        helpers.check_logits(got[None], helpers.plain_logits(folders[name], tuple(text), dtype)[-1:], dtype, what)

    for turn, sizes in enumerate([(5, 1, 12), (2, 9, 3), (1, 6, 4)]):
        trees = [tree(n, 10 * turn + n) for n in sizes]
        tokens = [rng.integers(0, V, n).tolist() for n in sizes]
        logits = engine.draft_step(slots, tokens, trees).float().cpu().numpy()
        row = 0
        paths = []
        for i, (toks, up) in enumerate(zip(tokens, trees)):
            for j in range(len(toks)):
                check(logits[row + j], texts[i] + [toks[k] for k in path_to(up, j)], "turn %d, sequence %d, node %d" % (turn, i, j))
            row += len(toks)
            paths.append(path_to(up, int(rng.integers(0, len(toks)))) if (turn, i) != (1, 0) else [])
        engine.keep(slots, paths)
        for i, path in enumerate(paths):
            texts[i] = texts[i] + [tokens[i][j] for j in path]
            assert engine.length(slots[i]) == len(texts[i])
        more = [[int(t)] for t in rng.integers(0, V, 3)]
        got = engine.step(slots, more).float().cpu().numpy()
        for i in range(3):
            texts[i] = texts[i] + more[i]
            check(got[i], texts[i], "the step behind turn %d, sequence %d" % (turn, i))
    engine.release(slots)
    assert all(g.pool.n_free == g.n_pages for g in engine.cache.kv_groups)


@pytest.mark.parametrize("filters", [{}, {"temperature": 0.9}, {"temperature": 0.8, "top_k": 20, "top_p": 0.9}, {"temperature": 1.1, "min_p": 0.05}])
@pytest.mark.parametrize("name", ["tiny_llama", "tiny_mistral", "tiny_llama3"])
def test_drafted_generation_gives_the_tokens_of_generate(folders, name, filters):
    """float32: the same tokens with trees of guesses as without, guessed from the text, by an oracle and by one that is always wrong;
    stop tokens end a request where they stand; the cache is whole again."""
    from yalm_amd import GenerationStats, generate, generate_drafted
    engine = engine_of(folders, name, torch.float32)
    V = tiny_configs.ALL[name]["vocab_size"]
    rng = np.random.default_rng(5)
    prompts = [(rng.integers(0, V, 4).tolist() * 6)[:n] for n in (2, 9, 21)] + [rng.integers(0, V, 5).tolist() for _ in range(4)]
    args = dict(max_new_tokens=24, seed=11, stop_ids=[], **{"temperature": 0.0, **filters})
    want = generate(engine, prompts, **args)
    assert generate_drafted(engine, prompts, **args) == want

    def oracle(history, n):
        which = next(i for i, p in enumerate(prompts) if history[:len(p)] == p and want[i][:len(history) - len(p)] == history[len(p):])
        ahead = (prompts[which] + want[which])[len(history) - 1:][:n]
        return ahead, list(range(-1, len(ahead) - 1))

    stats = GenerationStats()
    assert generate_drafted(engine, prompts, guess=oracle, max_nodes=5, stats=stats, batch_size=1, **args) == want
    assert stats.decode_steps < stats.new_tokens / 2 and stats.new_tokens == sum(map(len, want))
    wrong = lambda history, n: ([history[-1]] + [0] * (n - 1), [-1] + [0] * (n - 1))  # noqa: E731
    assert generate_drafted(engine, prompts, guess=wrong, max_nodes=3, **args) == want
    stop = want[1][5]
    cut = generate(engine, prompts, **{**args, "stop_ids": [stop]})
    assert generate_drafted(engine, prompts, guess=oracle, max_nodes=7, **{**args, "stop_ids": [stop]}) == cut
    assert not engine.cache.slots.held and all(g.pool.n_free == g.n_pages for g in engine.cache.kv_groups)


def test_drafted_generation_up_to_the_end_of_the_context(folders):
    from yalm_amd import generate, generate_drafted
    engine = engine_of(folders, "tiny_llama", torch.float32, max_tokens=128, max_batch=1)
    prompt = [3, 9, 4] * 30
    want = generate(engine, [prompt], max_new_tokens=100, stop_ids=[])
    assert len(want[0]) == engine.n_positions - len(prompt)
    assert generate_drafted(engine, [prompt], max_new_tokens=100, stop_ids=[], max_nodes=16) == want


@pytest.mark.parametrize("name", ["tiny_llama", "tiny_mistral"])
def test_filters_in_the_generation_loop(folders, name):
    """Tokens are the definition's picks from the plain implementation's logits."""
    from yalm_amd import generate
    from yalm_amd.sampling import uniform
    engine = engine_of(folders, name, torch.float32)
    prompt = [7, 100, 31, 5]
    got = generate(engine, [prompt], max_new_tokens=12, temperature=0.7, top_k=30, top_p=0.8, min_p=0.01, seed=5, stop_ids=[])[0]
    assert generate(engine, [prompt], max_new_tokens=12, temperature=0.7, top_k=30, top_p=0.8, min_p=0.01, seed=5, stop_ids=[], ahead=False)[0] == got
    cfg, w = R.read_folder(folders[name])
    agree = 0
    for step in range(12):
        logits = R.forward(w, cfg, prompt + got[:step])[-1].float().numpy()
        agree += sample_reference(logits, uniform(5, 0, step), 0.7, 30, 0.8, 0.01)[0] == got[step]
    assert agree >= 11                                         # a number may lie within the logits' rounding of a border
    greedy = generate(engine, [prompt], max_new_tokens=6, stop_ids=[])
    assert generate(engine, [prompt], max_new_tokens=6, top_k=5, top_p=0.5, stop_ids=[]) == greedy
    assert generate(engine, [prompt], max_new_tokens=6, temperature=2.0, top_k=1, stop_ids=[]) == greedy


def test_settings_for_each_row_and_their_refusals():
    from yalm_amd import Sampler
    logits = torch.randn((4, 500), generator=torch.Generator().manual_seed(1)).to("cuda:0")
    s = Sampler(3)
    one = [s.sample(logits[i:i + 1], t, [i], [2], top_k=k, top_p=p, min_p=m)[0]
           for i, (t, k, p, m) in enumerate([(0.0, 3, 0.5, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 9, 1.0, 0.1), (1.2, 0, 1.0, 0.0)])]
    every = s.sample(logits, [0.0, 0.7, 1.0, 1.2], range(4), [2] * 4, top_k=[3, 0, 9, 0], top_p=[0.5, 0.9, 1.0, 1.0], min_p=[0.0, 0.0, 0.1, 0.0])
    assert every == one and one[0] == int(logits[0].argmax())
    for bad in ({"top_p": 1.5}, {"min_p": -0.1}, {"top_k": -1}, {"top_k": [1, 2]}, {"top_p": float("nan")}):
        with pytest.raises(ValueError):
            s.sample(logits, 0.7, range(4), [0] * 4, **bad)
    with pytest.raises(ValueError):
        s.sample(logits, -1.0, range(4), [0] * 4, top_k=3)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", NAMES)
def test_several_answers_to_a_prompt(folders, name, dtype):
    """samples=n gives what n requests of the same prompt give, each from its own number; forks and the sequence they came from then go
    on independently."""
    from yalm_amd import GenerationStats, generate
    engine = engine_of(folders, name, helpers.torch_dtype(dtype), max_batch=7)
    V = tiny_configs.ALL[name]["vocab_size"]
    prompts = [np.random.default_rng(n).integers(0, V, n).tolist() for n in (3, 40, 8)]
    stats = GenerationStats()
    got = generate(engine, prompts, max_new_tokens=10, temperature=0.9, seed=4, stop_ids=[], samples=3, stats=stats)
    assert len(got) == 9 and stats.new_tokens == 90 and stats.prompt_tokens < 3 * sum(map(len, prompts))
    if dtype == "float32":
        assert got == generate(engine, [p for p in prompts for _ in range(3)], max_new_tokens=10, temperature=0.9, seed=4, stop_ids=[])
    assert not engine.cache.slots.held and all(g.pool.n_free == g.n_pages for g in engine.cache.kv_groups)


CARRYING = {"zebivik": zebivik_configs, "gemepel": gemepel_configs, "bovozen": bovozen_configs}


@pytest.mark.parametrize("design", sorted(CARRYING))
def test_forks_of_designs_that_carry_state(design):
    """A fork's logits are bit for bit those of the sequence it came from, and trees are refused."""
    from yalm_amd import Engine, Model, StepError
    cfg = next(v for k, v in vars(CARRYING[design]).items() if k.isupper() and isinstance(v, dict) and "layers" in v)
    engine = Engine(Model.random(cfg, 3, dtype=torch.float32), max_tokens=1024, max_batch=4)
    (s,) = engine.start(1)
    engine.step([s], [[5, 9, 2, 7, 1, 3, 8]])
    engine.step([s], [[4]])
    new = engine.fork(s, 2)
    for tok in (6, 1, 9):
        logits = [engine.step([x], [[tok]]).clone() for x in [s] + new]
        assert torch.equal(logits[0], logits[1]) and torch.equal(logits[0], logits[2])
    a, b = (engine.step([x], [[t]]).clone() for x, t in zip(new, (2, 3)))
    assert not torch.equal(a, b)
    with pytest.raises(StepError, match="drafted"):
        engine.draft_step([s], [[1, 2]])


def test_refused_drafts(folders):
    from yalm_amd import Engine, Model, StepError
    engine = engine_of(folders, "tiny_mistral", torch.float32, max_draft=6)
    a, b = engine.start(2)
    with pytest.raises(StepError, match="after its prompt"):
        engine.draft_step([a], [[1, 2]])
    engine.step([a, b], [[1, 2, 3], [4]])
    for tokens, parents, match in ([[1] * 7], None, "drafted tokens"), ([[]], None, "drafted tokens"), ([[1, 400]], None, "vocabulary"), \
            ([[1, 2, 3]], [[-1, 0, 2]], "parent"), ([[1, 2]], [[-1]], "parent"), ([[1], [2]], None, "same length"):
        with pytest.raises(StepError, match=match):
            engine.draft_step([a], tokens, parents)
    with pytest.raises(StepError, match="no drafted"):
        engine.keep([a], [[0]])
    engine.draft_step([a], [[1, 2, 3]], [[-1, 0, 0]])
    for path in ([1], [0, 1, 2], [0, 3], [0, 0]):
        with pytest.raises(StepError, match="path"):
            engine.keep([a], [path])
    for call in (lambda: engine.step([a], [[1]]), lambda: engine.draft_step([a], [[1]]), lambda: engine.fork(a, 1)):
        with pytest.raises(StepError, match="drafted"):
            call()
    engine.step([b], [[1]])
    with pytest.raises(StepError, match="one path"):
        engine.keep([a, a], [[0], [0]])
    engine.keep([a], [[0, 2]])
    engine.step([a], [[1]])
    engine.draft_step([a], [[1, 2]])
    engine.release([a])                                        # a sequence may end with its drafts undecided
    (c,) = engine.start(1)
    engine.step([c], [[5, 6]])
    assert Engine(engine.model, max_tokens=512).max_draft == 0
    sinks = Engine(Model.from_folder(folders["tiny_llama"], dtype=torch.float32, device="cuda:0", context=20), max_tokens=512, max_draft=4)
    (s,) = sinks.start(1)
    sinks.step([s], [[1, 2, 3]])
    with pytest.raises(StepError, match="sinks"):
        sinks.draft_step([s], [[1, 2]])


def test_the_command_line_samples_and_drafts(folders, capsys):
    from yalm_amd import generate
    from yalm_amd.cli import main
    engine = engine_of(folders, "tiny_llama", torch.float32)
    prompt = [1, 5, 17, 1, 5]
    args = [folders["tiny_llama"], "--tokens", "1,5,17,1,5", "-n", "7", "--dtype", "float32", "--seed", "3"]

    def run(*more):
        main(args + list(more))
        return capsys.readouterr().out

    filters = dict(temperature=0.8, top_k=30, top_p=0.9, seed=3)
    flags = ["-t", "0.8", "--top-k", "30", "--top-p", "0.9"]
    stop = [2]
    want = generate(engine, [prompt], max_new_tokens=7, stop_ids=stop, samples=2, **filters)
    out = run(*flags, "--samples", "2")
    assert all("[%d] %s\n" % (i, " ".join(map(str, w))) in out for i, w in enumerate(want))
    want = generate(engine, [prompt], max_new_tokens=7, stop_ids=stop, **filters)[0]
    assert " ".join(map(str, want)) in run(*flags, "--draft", "4")
    with pytest.raises(SystemExit):
        main(args + ["--draft", "4", "-T", "16"])


def test_settings_of_any_kind_of_number():
    """Python's numbers, numpy's, arrays, tensors: one for all rows or one for each, the same tokens."""
    from yalm_amd.sampling import Sampler
    logits = torch.randn((3, 900), generator=torch.Generator().manual_seed(2)).to("cuda:0") * 3
    sampler, ids, steps = Sampler(4), [0, 1, 2], [5, 6, 7]
    plain = sampler.sample(logits, 0.75, ids, steps)
    greedy = sampler.sample(logits, 0.0, ids, steps)
    assert sampler.sample(logits, np.float32(0.75), ids, steps) == plain == sampler.sample(logits, torch.tensor(0.75), ids, steps)
    assert sampler.sample(logits, np.float32(0.0), ids, steps) == greedy == sampler.sample(logits, 0, ids, steps)
    want = sampler.sample(logits, 0.75, ids, steps, top_k=20, top_p=0.5)
    for top_k in (np.int64(20), [20] * 3, np.full(3, 20), torch.full((3,), 20)):
        for top_p in (np.float64(0.5), (0.5, 0.5, 0.5), np.full(3, 0.5, np.float32), torch.tensor(0.5)):
            assert sampler.sample(logits, np.float32(0.75), ids, steps, top_k=top_k, top_p=top_p) == want
    assert sampler.sample(logits, np.zeros(3), ids, steps) == greedy
    for bad in (dict(top_k=[1, 2]), dict(top_p=1.5), dict(min_p=-0.1), dict(top_k=np.array([-1, 0, 0])), dict(top_p=float("nan"))):
        with pytest.raises(ValueError, match=next(iter(bad))):
            sampler.sample(logits, 1.0, ids, steps, **bad)


def test_guesses_deeper_than_the_window(folders):
    from yalm_amd import generate, generate_drafted
    engine = engine_of(folders, "tiny_mistral", torch.float32, max_draft=40)
    assert engine.max_draft_depth == tiny_configs.ALL["tiny_mistral"]["sliding_window"] < 40
    prompt = [5, 9] * 20
    chain = lambda history, n: ((history[-1:] + prompt * 2)[:n], list(range(-1, n - 1)))  # noqa: E731
    want = generate(engine, [prompt], max_new_tokens=60, stop_ids=[])
    assert generate_drafted(engine, [prompt], max_new_tokens=60, stop_ids=[], max_nodes=40, guess=chain) == want
    assert generate_drafted(engine, [prompt], max_new_tokens=60, stop_ids=[], max_nodes=40) == want


def test_draws_of_one_sampler_on_two_streams():
    """Draws under filters that may run at the same time: the tokens of draws one behind the other."""
    from yalm_amd.sampling import Sampler
    g = torch.Generator().manual_seed(6)
    logits = [(torch.randn((24, 50000), generator=g) * 2).to("cuda:0") for _ in range(4)]
    ids, how = list(range(24)), dict(top_p=0.9)
    sampler = Sampler(9)
    want = [sampler.sample(x, 0.8, ids, [i] * 24, top_k=[0, 40] * 12, **how) for i, x in enumerate(logits)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        drawn = []
        for i, x in enumerate(logits):
            with torch.cuda.stream(streams[i % 2]):
                drawn.append(sampler.draw(x, 0.8, ids, [i] * 24, top_k=[0, 40] * 12, **how))
        assert [d.tolist() for d in drawn] == want


def test_draws_behind_refused_ones():
    """A refused draw, then more draws than there are buffers, each read only when no more may be unread."""
    from yalm_amd.sampling import Sampler
    logits = [torch.randn((3, 700), generator=torch.Generator().manual_seed(i)).to("cuda:0") for i in range(9)]
    ids = [0, 1, 2]
    want = [Sampler(5).sample(x, 0.9, ids, [i] * 3, top_p=0.8) for i, x in enumerate(logits)]
    for refusals in (1, 2, 3):
        s, waiting, got = Sampler(5), [], []
        for i, x in enumerate(logits):
            if i < refusals:
                with pytest.raises(ValueError):
                    s.draw(x, 0.9, ids, [i] * 3, top_p=1.5)
            waiting.append(s.draw(x, 0.9, ids, [i] * 3, top_p=0.8))
            if len(waiting) == Sampler.HOST_BUFFERS:
                got.append(waiting.pop(0).tolist())
        assert got + [d.tolist() for d in waiting] == want


@pytest.mark.parametrize("window,max_tokens,max_nodes", [(64, 512, 16), (64, 64, 16), (63, 128, 20), (40, 64, 9), (200, 128, 5)])
def test_drafted_generation_to_the_end_where_a_window_is_as_long_as_the_context(folders, window, max_tokens, max_nodes):
    """Trees near the end of the context lie behind it, or are cut where the pages end: the tokens are generate()'s, by guesses that are
    right, by ones that are wrong and by the text's own."""
    from yalm_amd import Engine, Model, generate, generate_drafted
    engine = Engine(Model.from_folder(folders["tiny_mistral"], dtype=torch.float32, device="cuda:0", window=window), max_tokens=max_tokens, max_batch=2, max_draft=20)
    limit = engine.n_positions
    assert limit == tiny_configs.ALL["tiny_mistral"]["max_position_embeddings"]
    prompt = [5, 9, 31] * 4
    want = generate(engine, [prompt], max_new_tokens=limit, stop_ids=[])
    assert len(prompt) + len(want[0]) == limit

    def oracle(history, n):
        ahead = (prompt + want[0])[len(history) - 1:][:n - 1] + [7]
        return ahead + [8] * (n - len(ahead)), list(range(-1, len(ahead) - 1)) + [0] * (n - len(ahead))

    wrong = lambda history, n: ([history[-1]] + [0] * (n - 1), [-1] + [0] * (n - 1))  # noqa: E731
    for guess in ({}, {"guess": oracle}, {"guess": wrong}):
        assert generate_drafted(engine, [prompt], max_new_tokens=limit, stop_ids=[], max_nodes=max_nodes, **guess) == want
    assert not engine.cache.slots.held and all(g.pool.n_free == g.n_pages for g in engine.cache.kv_groups)


def test_what_outgrows_a_window_s_pages_is_refused(folders):
    """Drafted tokens that would lie on keys in sight, and a plain step that would: nothing changes, and what fits goes on."""
    from yalm_amd import Engine, Model, StepError
    engine = Engine(Model.from_folder(folders["tiny_mistral"], dtype=torch.float32, device="cuda:0", window=100), max_tokens=64, max_batch=1, max_draft=20, positions=200)
    (s,) = engine.start(1)
    engine.step([s], [list(range(3, 60))])
    with pytest.raises(StepError, match="window"):
        engine.draft_step([s], [[1] * 8])
    engine.draft_step([s], [[1] * 7])
    engine.keep([s], [[0, 1, 2, 3, 4, 5, 6]])
    assert engine.length(s) == 64
    for call in (lambda: engine.step([s], [[1]]), lambda: engine.draft_step([s], [[1]])):
        with pytest.raises(StepError, match="window"):
            call()
    engine.release([s])


def test_drafts_of_a_full_batch_stay_within_a_step_s_limit(folders):
    """An engine whose steps take few elements: trees are cut to a share of them, where a step was refused behind the prompts."""
    from yalm_amd import StepError, generate, generate_drafted
    engine = engine_of(folders, "tiny_mistral", torch.float32)
    widest = max(engine._widest_row, engine.model.vocab_size)
    prompts = [[7, 3, 9, 7, 3], [5, 6, 5, 6], [11] * 6, [2, 4, 8, 2, 4]]
    want = generate(engine, prompts, max_new_tokens=20, stop_ids=[])
    wide = lambda history, n: ([history[-1]] + [0] * (n - 1), [-1] + [0] * (n - 1))  # noqa: E731
    engine.MAX_ELEMENTS = 24 * widest + 1
    assert engine.max_step_drafts == 24
    assert generate_drafted(engine, prompts, max_new_tokens=20, stop_ids=[], max_nodes=20, guess=wide) == want
    assert generate_drafted(engine, prompts, max_new_tokens=20, stop_ids=[], max_nodes=20) == want
    slots = engine.start(2)
    engine.step(slots, [[1], [2]])
    with pytest.raises(StepError, match="25 drafted"):
        engine.draft_step(slots, [[1] * 20, [1] * 5], [[-1] + [0] * 19, [-1] + [0] * 4])
    engine.draft_step(slots, [[1] * 20, [1] * 4], [[-1] + [0] * 19, [-1] + [0] * 3])
    engine.release(slots)


@pytest.mark.parametrize("how", [{"context": 24}, {"window": 22}])
def test_texts_that_run_past_the_cache_s_tokens(folders, how):
    """A window's ring holds a text however long it runs: a few pages serve for hundreds of tokens, with drafts and without."""
    from yalm_amd import Engine, Model, generate, generate_drafted
    model = Model.from_folder(folders["tiny_mistral"], dtype=torch.float32, device="cuda:0", **how)
    prompts, n_new = [[1, 17, 200, 33, 5], [5, 9] * 40], 300
    at = dict(positions=400, max_batch=2, max_draft=9)
    args = dict(max_new_tokens=n_new, stop_ids=[])
    want = generate(Engine(model, max_tokens=1024, **at), prompts, **args)
    assert [len(w) for w in want] == [n_new] * 2
    small = Engine(model, max_tokens=256, **at)
    assert generate(small, prompts, **args) == want
    if "window" in how:
        assert generate_drafted(small, prompts, max_nodes=9, **args) == want
    assert all(g.pool.n_free == g.n_pages for g in small.cache.kv_groups)


def test_the_command_line_runs_a_text_past_its_context(folders, capsys):
    from yalm_amd import Engine, Model, generate
    from yalm_amd.cli import main
    model = Model.from_folder(folders["tiny_mistral"], dtype=torch.float32, device="cuda:0", context=24)
    want = generate(Engine(model, max_tokens=1024, positions=700), [[1, 17, 200]], max_new_tokens=500, stop_ids=[])[0]
    main([folders["tiny_mistral"], "--tokens", "1,17,200", "-n", "500", "-t", "0", "-T", "24", "--dtype", "float32"])
    stop = tiny_configs.ALL["tiny_mistral"].get("eos_token_id")
    assert " ".join(map(str, want[:want.index(stop) + 1] if stop in want else want)) in capsys.readouterr().out


@pytest.mark.parametrize("name,changes,max_tokens,seed", [("tiny_llama3", {}, 640, 1), ("tiny_llama3", {}, 1280, 2), ("tiny_mistral", {"sliding_window": 70, "max_position_embeddings": 300}, 1280, 3),
                                                         ("tiny_mistral", {"sliding_window": 100, "max_position_embeddings": 128}, 640, 4),
                                                         ("tiny_mistral", {"sliding_window": 150, "max_position_embeddings": 300}, 128, 5)])
def test_random_use_of_prompts_steps_trees_and_forks(tmp_path, name, changes, max_tokens, seed):
    """Sequences that start, go on by a token or a tree, keep any path of it, fork and end, in any order, in a cache that is often full:
    every logit is that of the sequence's own text, and what is refused changes nothing."""
    from yalm_amd import Engine, Model, StepError
    cfg = {**tiny_configs.ALL[name], **changes}
    folder = helpers.make_folder(tmp_path, name, cfg, seed=8)
    engine = Engine(Model.from_folder(folder, dtype=torch.float32, device="cuda:0"), max_tokens=max_tokens, max_batch=5, max_draft=24)
    rng = np.random.default_rng(seed)
    V, depth = cfg["vocab_size"], engine.max_draft_depth
    texts, done, refused = {}, {}, 0

    def books():
        return list(engine.cache.seq_len), sorted(engine.cache.slots.held), [(g.pool.n_free, g.table_host.tolist()) for g in engine.cache.kv_groups]

    def check(logits, text, what):
        helpers.check_logits(logits.float().cpu().numpy()[None], helpers.plain_logits(folder, tuple(text), "float32")[-1:], "float32", what)

    for turn in range(110):
        kind = rng.choice(["start", "step", "step", "tree", "tree", "tree", "fork", "end"], p=[0.12, 0.1, 0.1, 0.18, 0.18, 0.18, 0.08, 0.06])
        some = [s for s in texts if rng.random() < 0.7] or list(texts)[:1]
        before = books()
        try:
            if kind == "start":
                n = int(rng.choice([1, 5, 63, 64, 65, 100, 120]))
                (s,) = engine.start(1)
                text = rng.integers(0, V, n).tolist()
                try:
                    check(engine.step([s], [text])[0], text, "turn %d: prompt of %d" % (turn, n))
                    texts[s] = text
                finally:
                    if s not in texts:
                        engine.release([s])
            elif kind == "step" and some:
                new = [[int(rng.integers(0, V))] for _ in some]
                logits = engine.step(some, new)
                for i, s in enumerate(some):
                    texts[s] = texts[s] + new[i]
                    check(logits[i], texts[s], "turn %d: step" % turn)
            elif kind == "tree" and some:
                sizes = [int(rng.integers(1, 25)) for _ in some]
                trees = [tree(n, turn + n) for n in sizes]
                tokens = [rng.integers(0, V, n).tolist() for n in sizes]
                logits = engine.draft_step(some, tokens, trees)
                row, paths = 0, []
                for i, s in enumerate(some):
                    for j in {0, sizes[i] - 1, int(rng.integers(0, sizes[i]))}:
                        check(logits[row + j], texts[s] + [tokens[i][k] for k in path_to(trees[i], j)], "turn %d: node %d" % (turn, j))
                    row += sizes[i]
                    paths.append(path_to(trees[i], int(rng.integers(0, sizes[i]))) if rng.random() < 0.9 else [])
                engine.keep(some, paths)
                for i, s in enumerate(some):
                    texts[s] = texts[s] + [tokens[i][j] for j in paths[i]]
            elif kind == "fork" and texts:
                s = list(texts)[int(rng.integers(0, len(texts)))]
                for t in engine.fork(s, int(rng.integers(1, 3))):
                    texts[t] = list(texts[s])
            elif kind == "end" and texts:
                s = list(texts)[int(rng.integers(0, len(texts)))]
                engine.release([s])
                del texts[s]
            else:
                continue
            done[kind] = done.get(kind, 0) + 1
        except (StepError, RuntimeError) as e:
            assert any(w in str(e) for w in ("pages", "slots", "position", "longest", "window")), e
            assert books()[:2] == before[:2] and [f for f, _ in books()[2]] == [f for f, _ in before[2]]
            refused += 1
            if texts and rng.random() < 0.5:                   # make room
                s = list(texts)[0]
                engine.release([s])
                del texts[s]
        assert all(engine.length(s) == len(t) for s, t in texts.items())
    assert refused > 0 and len(done) == 5 and depth >= 24, (done, refused)
    engine.release(list(texts))
    assert all(g.pool.n_free == g.n_pages for g in engine.cache.kv_groups)
