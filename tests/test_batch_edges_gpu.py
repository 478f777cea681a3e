"""The batch operators where a user meets their edges.  References and bounds are those of test_batch_gpu
(64 bits, derived there from the formulas)."""

import math

import numpy as np
import pytest
import torch

from test_batch_gpu import BF, FP, I8, _batch, _check, _cu, _dense, _fast_reference, _gen, _plan_by_hand, _want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kernels(native):
    import asdsl_b200.kernels as k

    return k


def test_graph_outlives_workspace_growth(kernels):
    """A captured decode step replays the same bits after larger calls have grown its workspace, and leaves memory that
    was allocated since alone."""
    lens = [9000, 70, 4000]
    q, cache, table, lens_t, _, _ = _batch(kernels, lens, [1, 1, 1], 6, 2, 64, 16, BF, BF)
    pages = table[0, :200].contiguous()
    ws = kernels.AttentionWorkspace()

    def step():
        return (*kernels.attention_paged(q, cache, table, lens_t, return_lse=True, workspace=ws),
                *kernels.attention_shared_prefix(q, cache, pages, 3200, table, lens_t, return_lse=True, workspace=ws))

    want = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    # many more requests and rows than before, on the same workspace
    n, m = 9000, 2
    many = torch.randn(n * m, 6, 64, device="cuda", generator=_gen(1)).to(BF)
    wide, long = table[:1].expand(n, -1), lens_t[:1].expand(n).contiguous()
    cu = torch.arange(0, n * m + 1, m, dtype=torch.int32, device="cuda")
    big = kernels.attention_paged(many, cache, wide[:, :4], long.clamp(max=64), cu, workspace=ws).clone()
    kernels.attention_shared_prefix(many, cache, pages, 64, wide[:, :4], long.clamp(max=64), cu, workspace=ws)
    # whatever the allocator has free now is taken and filled
    fill = [torch.full((1 << 20,), 0x5A5A5A5A, dtype=torch.int32, device="cuda") for _ in range(64)]
    for _ in range(3):
        for t in got:
            t.fill_(7)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        again = kernels.attention_paged(many, cache, wide[:, :4], long.clamp(max=64), cu, workspace=ws)
        assert torch.equal(again, big)
    assert all((t == 0x5A5A5A5A).all() for t in fill)


@pytest.mark.parametrize("prefix", [False, True])
def test_capture_without_a_workspace(kernels, prefix):
    """A call that brings no workspace can be captured, and the graph keeps what it needs whatever is called after it."""
    lens, news = [3000, 70, 400], [1, 40, 2]
    q, cache, table, lens_t, cu, _ = _batch(kernels, lens, news, 6, 2, 64, 16, BF, BF)
    pages = table[0, :4].contiguous()

    def step():
        if prefix:
            return kernels.attention_shared_prefix(q, cache, pages, 64, table, lens_t, cu, return_lse=True)
        return kernels.attention_paged(q, cache, table, lens_t, cu, return_lse=True)

    want = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for _ in range(3):
        out.fill_(7), lse.fill_(7)
        graph.replay()
        step()  # eagerly between replays
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("n,page,new_max,tokens", [(3, 16, 1, 3), (40, 16, 30, 1200), (700, 64, 200, 140000), (1, 1, 5, 8)])
def test_plan_fed_with_its_own_totals(kernels, n, page, new_max, tokens):
    """A step's total_lens as the next step's kv_lens, over page boundaries and with many CTAs."""
    r = np.random.default_rng(n)
    kv, width = [0] * n, 2 + 8 * new_max // page
    table = [[-1] * width for _ in range(n)]
    plan = kernels.StepPlan(n, tokens, width, page)
    lens = _cu(kv)
    for step in range(8):
        new = r.integers(0, new_max + 1, n).tolist()
        free = (r.permutation(n * width) + step * n * width).tolist()
        want = _plan_by_hand(kv, new, free, table, page, width, tokens)
        kernels.plan_step(plan, lens, _cu(new), _cu(free))
        got = (plan.block_table, plan.cu_q, plan.total_lens, plan.slots, plan.positions, plan.requests, plan.counts)
        for name, g, w in zip(("table", "cu", "total", "slots", "positions", "requests", "counts"), got, want):
            assert g.tolist() == w, (step, name)
        kv, table, lens = want[2], want[0], plan.total_lens
        if step == 5 and n > 2:
            n -= 1  # the last request leaves
            kv, table, lens = kv[:n], table[:n], lens[:n]
    with pytest.raises(ValueError, match="overlap"):
        kernels.plan_step(plan, lens, plan.cu_q[:n], _cu(free))


def test_plan_flags_one_request_that_outgrows_the_table(kernels):
    """The flag comes from whichever thread meets the request, the same in every launch."""
    plan = kernels.StepPlan(900, 900, 2, 16)
    new, free = _cu([1] * 900), _cu(list(range(2000)))
    for b in (0, 31, 511, 512, 899):
        kv = torch.zeros(900, dtype=torch.int32, device="cuda")
        kernels.plan_step(plan, kv, new, free)
        assert plan.counts.tolist() == [900, 900, 0]
        kv[b] = 32
        for _ in range(20):
            kernels.plan_step(plan, kv, new, free)
            assert plan.counts.tolist() == [899, 900, 2]


@pytest.mark.parametrize("m,window,sinks", [(1, 50, 0), (1, 36, 0), (1, 30, 2), (4, 0, 0), (4, 60, 3), (60, 0, 0), (60, 45, 2), (60, 100, 0)])
@pytest.mark.parametrize("cache_dtype", [BF, I8])
def test_attention_table_narrower_than_the_lengths(kernels, m, window, sinks, cache_dtype):
    """Positions come from kv_lens; keys past the table's last page are unseen."""
    q, cache, table, lens_t, cu, _ = _batch(kernels, [100, 50], [m, m], 6, 2, 128, 16, BF, cache_dtype, with_cu=True)
    table = table[:, :4].contiguous()  # 64 positions
    out, lse = kernels.attention_paged(q, cache, table, lens_t, cu, window=window, sinks=sinks, return_lse=True)
    want = []
    for b, n in enumerate((100, 50)):
        k, v = _dense(cache, table[b, : -(-min(n, 64) // 16)], min(n, 64))
        want.append(_fast_reference(q[b * m : b * m + m].double(), k, v, n - m, window, sinks, 1 / math.sqrt(128)))
    _check(out, lse, tuple(torch.cat(x) for x in zip(*want)), BF)


@pytest.mark.parametrize("m", [1, 60])
def test_attention_windows_of_any_size(kernels, m):
    """The largest windows and sinks with more rows than keys (positions before key 0) stay within 32 bits."""
    q, cache, table, lens_t, cu, _ = _batch(kernels, [40, 3], [m, m], 6, 2, 64, 16, BF, BF, with_cu=True)
    want = kernels.attention_paged(q, cache, table, lens_t, cu, return_lse=True)
    for window, sinks in ((2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (2**31 - 30, 5), (1, 2**31 - 1)):
        got = kernels.attention_paged(q, cache, table, lens_t, cu, window=window, sinks=sinks, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (window, sinks)


def _far_apart(kernels, m, dtype, cache_dtype, dim, n, copies, outlier):
    """`copies` requests (enough that none is split over CTAs) of m rows of ones on the same n keys: all scores 0 but
    of key 5, 17.6 above them and with a value of 0, or (outlier) 60 below them and with values 2^21 times the others'."""
    q, cache, table, lens_t, _, _ = _batch(kernels, [n], [m], 6, 2, dim, 64, dtype, cache_dtype, with_cu=True)
    score = (-60.0 if outlier else 17.6) / (dim * dim**-0.5)
    page, at = table[0, 0].long(), 5
    cache.k.zero_()
    if cache_dtype == I8:
        cache.k[page, at] = 127 if score > 0 else -127
        cache.k_scales.fill_(abs(score) / 127)
        cache.v.copy_(cache.v.abs().clamp(min=1))
        cache.v_scales.fill_(0.01)
    else:
        cache.k[page, at] = score
        cache.v.copy_(cache.v.abs())
    if outlier:
        cache.v_scales[page, at] = 0.01 * 2**21
    else:
        cache.v[page, at] = 0
    q.fill_(1.0)
    scale = dim**-0.5
    out, lse = kernels.attention_paged(q.repeat(copies, 1, 1), cache, table.expand(copies, -1), lens_t.expand(copies).contiguous(),
                                       _cu(list(range(0, copies * m + 1, m))), scale=scale, return_lse=True)
    want = tuple(x.repeat(copies, *(1,) * (x.dim() - 1)) for x in _want(q, cache, table, [n], [m], 64, 0, 0, scale))
    _check(out, lse, want, dtype, str((m, dtype, cache_dtype, dim)))


# few rows, and enough for the many-rows kernel
@pytest.mark.parametrize("m,copies", [(1, 400), (5, 400), (40, 80)])
@pytest.mark.parametrize("dtype,cache_dtype,dim", [(FP, FP, 64), (FP, FP, 128), (BF, I8, 128), (FP, I8, 64), (FP, I8, 128), (BF, BF, 64)])
def test_attention_long_low_tail(kernels, m, copies, dtype, cache_dtype, dim):
    """Weights 2^25 below the largest carry the output where the largest one's value is 0: they keep their bits."""
    _far_apart(kernels, m, dtype, cache_dtype, dim, 30000, copies, False)


@pytest.mark.parametrize("m,copies", [(1, 400), (5, 400), (40, 80)])
@pytest.mark.parametrize("dtype,dim", [(BF, 128), (FP, 64), (FP, 128)])
def test_attention_value_scale_far_above_the_others(kernels, m, copies, dtype, dim):
    """An int8 key of no weight whose V scale is 2^21 times the others' does not cost them their bits."""
    _far_apart(kernels, m, dtype, I8, dim, 700, copies, True)


@pytest.mark.parametrize("m", [1, 2, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_query_elements_far_apart(kernels, m, dim):
    """bf16 queries on int8 pages: elements 2^20 below the row's largest count when that one meets codes of 0."""
    q, cache, table, lens_t, cu, _ = _batch(kernels, [300], [m], 6, 2, dim, 16, BF, I8, with_cu=True)
    q[..., 3] = 2.0**20
    cache.k[..., 3] = 0
    out, lse = kernels.attention_paged(q, cache, table, lens_t, cu, return_lse=True)
    _check(out, lse, _want(q, cache, table, [300], [m], 16, 0, 0, dim**-0.5), BF)


@pytest.mark.parametrize("size", [2.0**-133, 2.0**-100, 2.0**-40, 2.0**60, 3e38])
def test_attention_query_rows_of_any_size(kernels, size):
    """bf16 query rows from subnormal to the largest on int8 pages: the scores are in proportion (scales of the keys make up
    for the size where the product has room)."""
    q, cache, table, lens_t, _, _ = _batch(kernels, [200], [1], 6, 2, 64, 16, BF, I8)
    q = q.clamp(-1, 1) * size
    cache.k_scales.copy_(cache.k_scales * min(1 / size, 2.0**100))
    out, lse = kernels.attention_paged(q, cache, table, lens_t, return_lse=True)
    _check(out, lse, _want(q, cache, table, [200], [1], 16, 0, 0, 1 / 8), BF)


# ---- the decoder of a batch -------------------------------------------------------------------------

PROMPTS = [[5, 9, 100, 7, 3], [1], [400, 2, 2, 31, 8, 99, 17, 250, 40, 12, 13, 14, 15, 16, 18, 19, 20, 21]]


@pytest.fixture(scope="module")
def model(native):
    from asdsl_b200.inference.synthetic import TINY, build_model

    return build_model(TINY, 11)


def test_prefix_with_a_window_is_refused(model):
    """The shared prefix is attended whole by every row: under a window that would be another rule than without it."""
    from asdsl_b200.inference.batch import BatchDecoder

    dec = BatchDecoder(model, 4, 64, page_size=16, window=6, sinks=2)
    with pytest.raises(ValueError, match="window"):
        dec.generate(PROMPTS, 2, prefix=[3, 77, 500])
    assert dec.taken == 0
    assert len(dec.generate(PROMPTS, 2)[0]) == len(PROMPTS[0]) + 2


def test_penalties_see_the_prefix(model):
    """The prefix's ids are part of each request's history, as if they stood in its prompt."""
    from asdsl_b200.inference.batch import BatchDecoder

    prefix = [3, 77, 500, 41, 6, 8]
    dec = BatchDecoder(model, 4, 64, page_size=16)
    plain, repeated, counted = [], [], []
    dec.generate(PROMPTS, 1, prefix=prefix, logits_out=plain)
    dec.reset()
    dec.generate(PROMPTS, 1, prefix=prefix, repetition=8.0, logits_out=repeated)
    dec.reset()
    dec.generate(PROMPTS, 1, prefix=prefix, frequency=3.0, presence=5.0, logits_out=counted)
    for b, p in enumerate(PROMPTS):
        x, y = plain[0][b], repeated[0][b]
        want = x.clone()
        ids = torch.tensor(sorted(set(prefix + p)), device="cuda")
        want[ids] = torch.where(x[ids] > 0, x[ids] / 8, x[ids] * 8)  # a power of two: exact
        assert torch.equal(y, want)
        assert torch.equal(counted[0][b], x)  # no output yet


def test_penalties_under_a_prefix_as_over_the_joined_prompts(model):
    """generate([p], prefix=P) and generate([P + p]) penalise the same ids and give the same logits (within the two
    attentions' rounding, re-quantized to 8 bits by each projection: 5e-2 of the logits' norm)."""
    from asdsl_b200.inference.batch import BatchDecoder

    prefix = [3, 77, 500, 41, 6, 8, 7, 3]
    dec = BatchDecoder(model, 4, 64, page_size=16)
    shared, joined = [], []
    dec.generate(PROMPTS, 1, prefix=prefix, repetition=8.0, logits_out=shared)
    dec.reset()
    dec.generate([prefix + p for p in PROMPTS], 1, repetition=8.0, logits_out=joined)
    x, y = shared[0].double(), joined[0].double()
    assert ((x - y).norm(dim=-1) <= 5e-2 * y.norm(dim=-1)).all()
