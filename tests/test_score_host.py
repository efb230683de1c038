"""gl3_forward_score's host code without a GPU: HIP's calls land in host memory (hip_on_host.py)."""
import hip_on_host


def test_a_score_whose_buffers_did_not_fit_is_asked_for_again():
    """Its own error alone: the next call, and any other call of the plan, does not report it again."""
    hip_on_host.run("""
    t, w, ids, f = np.arange(4, dtype=np.int32), np.zeros(1, np.int32), np.zeros(4, np.int32), np.zeros(200, np.float32)
    p = lambda a: a.ctypes.data
    score = lambda: L.gl3_forward_score(ctx, 0, p(t), 4, 0, p(w), 1, p(ids), 2, p(f), p(ids), p(f), p(ids), p(f))
    step = lambda: L.gl3_forward_step(ctx, 0, p(t), 4, 0, p(w), 1, p(f))
    for fails in (fake.fake_fail_malloc, fake.fake_fail_host_malloc):          # scratch; targets and results
        for again in (score, step):
            ctx = tiny_plan(max_batch=8)
            assert L.gl3_finalize(ctx) == 0, L.gl3_last_error(ctx)
            fails(1)
            assert score() == hip.E_OOM and fake.fake_pending() == 0
            assert again() == 0, L.gl3_last_error(ctx)
            assert score() == 0, L.gl3_last_error(ctx)
            L.gl3_destroy(ctx)
    """)
