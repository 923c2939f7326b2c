"""Generation that drafts: instead of one token a step every sequence goes on by a tree of guesses, the model says in one step what
it would have drawn behind each of them, and the path of guesses that it agrees with is kept, with the token behind it.

The tokens are those of generate() with the same seed, up to rounding: the token of a place is drawn from the model's own logits there, with
the number that belongs to the request and the place, and a guess is kept only if it is that token.  A guesser that is never right
costs a step of wider rows a token, launched kernel by kernel, and its own time on the host; each guess that is right saves a step.  At the Mistral-7B
shape in bfloat16, 8 nodes, tokens a second behind 3,000 tokens: one sequence 254 with the text's own guesses where none is right and 2,227 with ones that
always are (generate: 362), eight sequences 1,120 where few are (2,440)."""
from .cache.manager import PAGE
from .generate import GenerationStats, plan_batches


def lookup_tree(history, n, longest=3, branches=3):
    """Guesses at what follows `history`, from history itself: what followed the places where its last tokens (the last `longest`, else
    fewer) stood before, the latest ones first.  Returns (tokens, parents) of a tree of at most n nodes whose root is history's last token.
    It looks through the whole text, up to three times: 0.5 ms for 3,000 tokens that say nothing, 4.6 for 28,000."""
    tokens, parents = [history[-1]], [-1]
    children = {}                                     # (node, token) -> node
    last = len(history) - 1
    found = []
    for size in range(min(longest, last), 0, -1):
        tail = history[last + 1 - size:]
        for at in range(last - size, -1, -1):
            if len(found) >= branches:
                break
            if history[at:at + size] == tail and at + size not in found:
                found.append(at + size)
        if found:
            break
    each = (n - 1) // max(1, len(found))
    for at in found:
        node = 0
        for tok in history[at:at + each]:
            if (node, tok) not in children:
                if len(tokens) >= n:
                    break
                children[node, tok] = len(tokens)
                tokens.append(tok)
                parents.append(node)
            node = children[node, tok]
    return tokens, parents


def accept(tokens, parents, drawn):
    """The walk down a tree: from the root to the child that the model drew behind it, and on.  Returns (the path's nodes, the tokens that
    the sequence goes on by: those of the path behind the root, and the one drawn behind its end)."""
    child = {(p, t): j for j, (p, t) in enumerate(zip(parents, tokens)) if j > 0}
    path, new = [0], [drawn[0]]
    while (path[-1], new[-1]) in child:
        path.append(child[path[-1], new[-1]])
        new.append(drawn[path[-1]])
    return path, new


def generate_drafted(engine, prompts, max_new_tokens=256, temperature=0.0, seed=0, stop_ids=None, batch_size=None, sampler=None, on_token=None,
                     stats=None, request_ids=None, top_k=0, top_p=1.0, min_p=0.0, max_nodes=8, guess=lookup_tree):
    """As generate() (without `ahead`: a step's tree hangs on the tokens of the step before).  guess(history, n): the (tokens, parents) of a tree
    of at most n nodes behind a request's prompt and new tokens, the root being the last of them."""
    from .sampling import Sampler
    from .sampling.sampler import filters_for_all, one_for_all
    sampler = sampler or Sampler(seed)
    filters = filters_for_all(top_k, top_p, min_p)
    if isinstance(sampler, Sampler):
        one_for_all("temperature", temperature)
    stats = stats if stats is not None else GenerationStats()
    stop = set(stop_ids if stop_ids is not None else getattr(engine.model.spec, "eos_token_ids", None) or [])
    ids = list(request_ids) if request_ids is not None else list(range(len(prompts)))
    max_len, max_nodes = engine.n_positions, int(max_nodes)
    if not 1 <= max_nodes <= engine.max_draft:
        raise ValueError("trees of %d nodes: the engine takes 1 to %d" % (max_nodes, engine.max_draft))
    results = [[] for _ in prompts]
    if max_new_tokens <= 0 or not prompts:
        return results

    def take(i, new):
        """Appends a request's new tokens up to its end; True if it goes on."""
        for tok in new:
            results[i].append(tok)
            stats.new_tokens += 1
            if on_token is not None:
                on_token(i, tok)
            n = len(results[i])
            if n >= max_new_tokens or len(prompts[i]) + n >= max_len or tok in stop:
                return False
        return True

    import time
    room = max_new_tokens + max_nodes                 # drafted tokens lie in the cache beside the kept ones
    for batch in plan_batches([len(p) for p in prompts], room, batch_size, engine.cache.n_pages * PAGE, engine.cache.n_slots, max_len,
                              engine.cache.whole_rings()):
        stats.batches += 1
        stats.batch_sizes.append(len(batch))
        slots = engine.start(len(batch))
        live, held = list(zip(batch, slots)), set(slots)
        try:
            t0 = time.perf_counter()
            logits = engine.step(slots, [prompts[i] for i in batch])
            stats.bytes_read += engine.step_bytes(slots)
            drawn = sampler.sample(logits, temperature, [ids[i] for i in batch], [0] * len(batch), **filters)
            stats.prefill_seconds += time.perf_counter() - t0
            stats.prompt_tokens += sum(len(prompts[i]) for i in batch)
            stats.batches_first_tokens += len(batch)
            t0 = time.perf_counter()
            live = [(i, s) for (i, s), tok in zip(live, drawn) if take(i, [tok])]
            while True:
                ended = held.difference(s for _, s in live)
                engine.release(sorted(ended))
                held.difference_update(ended)
                if not live:
                    break
                trees = []
                share = min(max_nodes, engine.max_step_drafts // len(live))       # of what one step takes
                for i, s in live:
                    history = list(prompts[i]) + results[i]
                    # no deeper than the request's tokens, the context and a window go, and no wider than the places behind its tokens
                    left = min(max_new_tokens - len(results[i]), max_len - len(history), engine.max_draft_depth)
                    tokens, parents = guess(history, max(1, min(share, max_len - engine.length(s), engine.cache.room(s))))
                    trees.append(_shallow(tokens, parents, left))
                running = [s for _, s in live]
                logits = engine.draft_step(running, [t for t, _, _ in trees], [p for _, p, _ in trees])
                stats.bytes_read += engine.step_bytes(running)
                stats.decode_steps += 1
                drawn = sampler.sample(logits, temperature, [ids[i] for (i, _), (t, _, _) in zip(live, trees) for _ in t],
                                       [len(results[i]) + d for (i, _), (_, _, depth) in zip(live, trees) for d in depth], **filters)
                at, paths, going = 0, [], []
                for (i, s), (tokens, parents, _) in zip(live, trees):
                    path, new = accept(tokens, parents, drawn[at:at + len(tokens)])
                    at += len(tokens)
                    paths.append(path)
                    if take(i, new):
                        going.append((i, s))
                engine.keep(running, paths)
                live = going
            stats.decode_seconds += time.perf_counter() - t0
        except BaseException:
            engine.release(sorted(held))              # a failed batch gives back what it still holds
            raise
    return results


def _shallow(tokens, parents, left):
    """(tokens, parents, depths) of the nodes that stand less than `left` deep (the root always)."""
    new, depths = {}, []
    kept_tokens, kept_parents = [], []
    for j, (tok, p) in enumerate(zip(tokens, parents)):
        d = 0 if j == 0 else depths[new[p]] + 1 if p in new else left
        if j > 0 and d >= left:
            continue
        new[j] = len(depths)
        depths.append(d)
        kept_tokens.append(tok)
        kept_parents.append(new[p] if j else -1)
    return kept_tokens, kept_parents, depths
