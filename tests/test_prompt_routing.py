"""The restated routing of prompt_ref.py by groups, without a GPU."""
import numpy as np

import prompt_ref


def test_a_group_that_is_kept_holds_its_best_expert():
    """(test_prompt_ops.py asks of the best group only whether it is a group.)"""
    rng = np.random.default_rng(3)
    logits, bias = rng.normal(size=(50, 12)), rng.normal(size=12) * 0.1
    ids, _ = prompt_ref.route(logits, 3, "sigmoid", bias, 4, 2, 2, True, 2.5)
    for t in range(50):
        c = 1 / (1 + np.exp(-logits[t])) + bias
        best = max(range(4), key=lambda g: sum(sorted(c[3 * g:3 * g + 3])[1:]))
        assert 3 * best + int(np.argmax(c[3 * best:3 * best + 3])) in ids[t]
