"""A plan with an 8-bit head whose gl3_finalize fails and is called again: the logits' multiplier reaches the final norm once.  Without a GPU: HIP's calls land in
host memory (hip_on_host.py)."""
import pytest

import hip_on_host


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("fails", [0, 1, 2, 3])
def test_finalize_is_called_again(fails, tied):
    hip_on_host.run("""
    MUL = 3.0
    norm = np.random.default_rng(2).uniform(1, 2, 64).astype(np.float32)
    ctx = tiny_plan(tied={tied}, flags=hip.FLAG_INT8_HEAD, norm=norm, logit_scale=MUL)
    fails = {fails}
    if fails:
        fake.fake_fail_malloc(fails)          # codes, scales, scratch
        assert L.gl3_finalize(ctx) != 0
        assert fake.fake_holds(norm.tobytes(), norm.nbytes) == 1 and fake.fake_pending() == 0
    assert L.gl3_finalize(ctx) == 0, L.gl3_last_error(ctx)
    once, twice = (norm * np.float32(MUL)).tobytes(), (norm * np.float32(MUL) * np.float32(MUL)).tobytes()
    assert fake.fake_holds(once, len(once)) == 1 and fake.fake_holds(twice, len(twice)) == 0
    assert L.gl3_finalize(ctx) == 0          # finalized: nothing happens
    assert fake.fake_holds(once, len(once)) == 1
    L.gl3_destroy(ctx)
    """.format(fails=fails, tied=tied))
