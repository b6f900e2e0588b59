"""CPU tests of how texts find the cached prompt they stand behind."""
import random
import threading

import abstracts_search_amd.sentence_transformers as st


def brute(cached, ids):
    best = (0, None)
    for key, handle in cached.items():
        if best[0] < len(key) < len(ids) and tuple(ids[:len(key)]) == key:
            best = (len(key), handle)
    return best


def test_the_longest_prompt_in_front():
    rng = random.Random(1)
    for trial in range(300):
        letters = rng.choice([2, 3, 40])
        ids = lambda n: [rng.randrange(letters) for _ in range(n)]
        keys = [tuple(ids(rng.randint(1, 9))) for _ in range(rng.randint(0, 30))]
        keys += [k + tuple(ids(rng.randint(1, 4))) for k in keys[::2]]          # prompts that begin as another one
        cached = st._Prompts({k: i for i, k in enumerate(keys)})
        for _ in range(60):
            text = list(rng.choice(keys)) + ids(rng.randint(0, 3)) if keys and rng.random() < 0.7 else ids(rng.randint(0, 12))
            assert cached.behind(text) == brute(cached, text), (keys, text)
    assert st._Prompts({(1, 2): 0}).behind([1, 2]) == (0, None)                 # nothing stands behind it
    import numpy as np
    assert st._Prompts({(1, 2): 0}).behind(np.array([1, 2, 3], np.int32)) == (2, 0)


def test_many_long_prompts_are_found_quickly():
    """two hundred prompts that differ at their ends: a lookup compares a few of them, not all"""
    class Counted(int):
        compared = 0

        def __eq__(self, other):
            Counted.compared += 1
            return int.__eq__(self, other)

        __hash__ = int.__hash__
    base = list(range(1000))
    cached = st._Prompts({tuple(base + [i] * 5): i for i in range(200)})
    text = [Counted(i) for i in base + [123] * 5 + [7, 8]]
    assert cached.behind(text) == (1005, 123)
    assert Counted.compared < 15 * 1010, Counted.compared                       # (bisection: 8 comparisons, and the last one's slice)


def test_lookups_beside_prompts_that_come():
    """a model's prompts are replaced, not changed: whoever looks one up meanwhile goes on with what there was"""
    model = st.SentenceTransformer.__new__(st.SentenceTransformer)
    model._cached_prompts, model._prompts_lock = st._Prompts(), threading.Lock()
    stop, errors = threading.Event(), []

    def look():
        try:
            while not stop.is_set():
                cached = model._cached_prompts
                for i in range(50):
                    n, h = cached.behind([i, 1, 2, 3])
                    assert (n, h) in ((0, None), (3, i))
        except Exception as e:                                                  # pragma: no cover
            errors.append(e)

    ts = [threading.Thread(target=look) for _ in range(3)]
    [t.start() for t in ts]
    for _ in range(20):
        for i in range(50):
            with model._prompts_lock:
                model._cached_prompts = st._Prompts({**model._cached_prompts, (i, 1, 2): i})
        with model._prompts_lock:
            model._cached_prompts = st._Prompts()
    stop.set()
    [t.join() for t in ts]
    assert not errors


def groups(texts, prompts, batch_size=None, **attrs):
    """{prompt's number or None: how many texts} of encode_tokens' passes; texts: [(prompt's number or None, tokens of its own)]"""
    model = st.SentenceTransformer.__new__(st.SentenceTransformer)
    for k, v in attrs.items():
        setattr(model, k, v)
    keys = [tuple([1000 + i] * n) for i, n in enumerate(prompts)]
    lists = [list(keys[p] if p is not None else ()) + [7] * own for p, own in texts]
    run, got = model._groups(lists, st._Prompts({k: i for i, k in enumerate(keys)}), batch_size)
    assert sorted(i for _, members in got for i in members) == list(range(len(texts)))          # each text once
    for handle, members in got:
        for i in members:
            assert run[i] == (lists[i] if handle is None else lists[i][len(keys[handle]):])
            assert handle is None or texts[i][0] == handle
    assert len({h for h, _ in got}) == len(got) and all(m for _, m in got)
    return {h: len(m) for h, m in got}


def test_one_text_behind_each_of_many_prompts_share_a_pass():
    """a pass a prompt would stream all the weights for each"""
    assert groups([(i, 5) for i in range(30)], [160] * 30) == {None: 30}
    assert groups([(i, 5) for i in range(2)], [160] * 2) == {0: 1, 1: 1}
    many = groups([(i, 60) for i in range(30) for _ in range(8)], [160] * 30)
    assert many == {i: 8 for i in range(30)}
    # a prompt with much behind it keeps its pass, the small ones go together, and with the texts behind none
    assert groups([(0, 50)] * 40 + [(i, 5) for i in range(1, 12)] + [(None, 30)], [400] + [160] * 11) == {0: 40, None: 12}
    assert groups([(i, 5) for i in range(30)], [160] * 30, prompt_pass_tokens=0) == {i: 1 for i in range(30)}
    assert groups([(i, 5) for i in range(5)], [4000] * 5) == {i: 1 for i in range(5)}
    assert groups([], []) == {}


def test_short_passes_are_judged_one_by_one():
    """forty queries of 31 tokens one at a time take the query-time path with their prompt's tokens, as one of them does"""
    assert groups([(0, 11)], [20]) == {None: 1}
    assert groups([(0, 11)] * 40, [20], batch_size=1) == {None: 40}
    assert groups([(0, 11)] * 40, [20]) == {0: 40}
    assert groups([(0, 11)] * 40, [20], batch_size=1, prompt_break_even=(0, 0, 0)) == {0: 40}
    assert groups([(0, 11)] * 40, [20], token_budget=None) == {0: 40}
    assert groups([(0, 29)] * 3, [20], batch_size=1) == {0: 3}
