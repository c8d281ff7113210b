"""The gated delta rule as a mixer in bfloat16 where a step holds decoded tokens, portions and whole prompts side by side, and in
decode steps of their own, every row against the plain implementation in 64 bits.

Tolerance: that of test_gpu_delta_mixer.py for a prompt's last row, here for every row: an activation is rounded to 8 bits
(2^-9.8 of it, the mean square) some nine times a layer, which three layers, each with a gain of a few, leave as one or two hundredths of the
largest logit, and the largest of 97 logits of 185 rows as about four times that: 0.08."""
import numpy as np
import pytest

import helpers
from test_gpu_delta_mixer import VOCAB, folders, plain_logits, runner_of, step  # noqa: F401  (folders: a fixture)

pytestmark = pytest.mark.gpu


def close(row, want):
    return np.abs(row - want).max() < 0.08 * np.abs(want).max()


@pytest.mark.parametrize("seed", [2, 3])
def test_every_row_of_mixed_steps(folders, seed):  # noqa: F811
    requests = {k: helpers.random_ids(VOCAB, n, i) for i, (k, n) in enumerate({"a": 75, "b": 9, "c": 40, "d": 61}.items())}
    wanted = {key: plain_logits(folders["wide"], ids).numpy() for key, ids in requests.items()}
    runner = runner_of(folders["wide"], "bfloat16")
    rows = helpers.run_trace_in_process(runner, helpers.trace_mixed(requests, seed=seed, max_live=3))
    assert len(rows) == 185
    for (key, pos), row in rows.items():
        assert close(row, wanted[key][pos])


def test_decode_steps_beside_prompts_and_alone(folders):  # noqa: F811
    folder = folders["wide"]
    runner = runner_of(folder, "bfloat16")
    ids = [helpers.random_ids(VOCAB, n, 20 + n) for n in (33, 5, 18)]
    handles = [runner.cache.open(i) for i in range(3)]
    for handle, own in zip(handles, ids):
        step(runner, (handle, own))
    for turn in range(6):
        fresh = [helpers.random_ids(VOCAB, 40 if turn == 2 and i == 1 else 1, 50 + 10 * turn + i) for i in range(3)]
        rows = step(runner, *zip(handles, fresh))
        for own, more, row in zip(ids, fresh, rows):
            own += more
            assert close(row, plain_logits(folder, own)[-1].numpy())
