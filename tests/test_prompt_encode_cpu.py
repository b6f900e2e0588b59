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
