"""The bounds of extend's one-launch form, on either side of each: 1024 entries, 32768 table entries, 4096 rows, 32768
state rows; against the restatement with loops."""
import numpy as np
import pytest

from tests.test_request_tables_gpu import i32, pair, same_state, same_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, R, width, total", [
    (64, 64, 512, 300), (64, 64, 513, 300), (63, 70, 521, 300), (1, 1, 32768, 5), (1, 1, 32769, 5),
    (1024, 1024, 32, 3000), (1024, 1024, 33, 3000), (1025, 1025, 8, 3000), (8, 8, 40, 4096), (8, 8, 40, 4097),
    (9, 32768, 40, 100), (9, 32800, 40, 100)])
def test_both_sides_of_the_one_launch_form(gpu, B, R, width, total):
    rng = np.random.RandomState(B + width + total)
    bs, held = 16, min(width, 12)
    t, m = pair(gpu, bs, R, width, rng.permutation(B * held + 400), num_blocks=B * held + 400)
    rows = rng.permutation(R)[:B]
    for _ in range(2):
        new = rng.multinomial(total - 3, np.ones(B) / B) if B <= 9 else rng.randint(0, 3, B)
        new = np.minimum(new, held * bs - m.requests[rows, 0])
        step = t.extend(i32(rows, gpu), i32(new, gpu), total_q=total, max_blocks_per_seq=width)
        want = m.extend(rows, new, width, total)
        same_step(step, want)
        same_state(t, m)
        kept = [rng.randint(0, n + 1) if n else 0 for n in new]
        lens = t.keep(i32(rows, gpu), step.context_lens, step.q_start_loc, i32(kept, gpu))
        assert lens.tolist() == m.keep(rows, want[1], want[2], kept).tolist()
        same_state(t, m)
    t.release(i32(rows, gpu))
    m.release(rows)
    same_state(t, m)
