"""Decode over a shared prefix in tables with room for gigabytes, where the kernels for shared pages run: whatever the number of sequences that share, the tolerances are those of
a plain step, as tests/test_paged_cache.py derives them (a probability is kept as two 16-bit numbers)."""
import pytest
import torch

import test_paged_conversations as conversations
from test_paged_cache import BF16, F16, _close, _ops
from test_paged_conversations import _int32, _shared_setup


def _wide_table(s, keys_and_values=1_000_000_000):
    """The setup's table with room for so many bytes of keys and values (zeros, which nothing reads), or for 2^20 keys a sequence."""
    pages = min(keys_and_values // (s.table.shape[0] * s.cache.page_size * s.hkv * s.d * 4) + 1, (1 << 20) // s.cache.page_size)
    return torch.cat([s.table, torch.zeros(s.table.shape[0], max(pages - s.table.shape[1], 0), dtype=torch.int32, device="cuda")], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefixes,sizes,own,hq,hkv,d,page,layout,alone", [
    ([40], [70], [17, 1, 0, 90], 28, 4, 128, 32, "part", []),
    ([9, 13, 1], [40, 1, 30], [33, 64], 32, 8, 64, 256, "heads", [1]),
    ([157], [33], [7, 1000], 8, 2, 128, 64, "heads", []),
    ([70], [33], [20, 0, 3], 32, 8, 128, 64, "rows", [5]),
    ([600], [9], [20], 71, 1, 64, 16, "heads", []),
    ([313], [3], [2], 8, 2, 128, 64, "rows", [900]),
    ([30], [5], [5000, 20], 71, 1, 64, 16, "heads", [3000]),
    ([40], [4], [0, 9000], 40, 2, 128, 32, "heads", []),
])
def test_shared_steps_are_as_precise_as_plain_ones(prefixes, sizes, own, hq, hkv, d, page, layout, alone, dtype):
    s, shared, groups = _shared_setup(prefixes, sizes, own, hkv, d, page, dtype, hq + page, layout, 0, alone)
    table, q = _wide_table(s), s.queries(hq)
    for scale in (d ** -0.5, 0.3, 0.004):
        _close(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups, sm_scale=scale), q, s, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("batch,hq,hkv,d", [(40, 8, 2, 128), (40, 8, 2, 64), (2, 8, 2, 128)])
def test_many_equal_keys_far_below_a_sink(batch, hq, hkv, d, dtype):
    """A key of 16 to 20 nats more than the 4096 others, whose values are zeros: the output is what these have together.  (At 20 nats a probability of fp16, kept as 2^15 times itself on a
    grid of 2^-24, is off by 2^-11.1 of it, which the rounding of scores, of up to 20, and of sums over 4096 keys covers.)"""
    s, shared, groups = _shared_setup([64], [batch], [1], hkv, d, 64, dtype, 7)
    s.cache.keys.zero_()
    s.cache.values.fill_(64.0)
    first = s.table[0, 0].long()
    s.cache.keys[first, :, 0, 0], s.cache.values[first, :, 0] = 16.0, 0.0
    q = torch.zeros(batch, hq, d, dtype=dtype, device="cuda")
    q[:, :, 0] = torch.linspace(1.0, 1.25, batch * hq, device="cuda").view(batch, hq).to(dtype)
    _close(_ops().paged_shared_decode_attention(s.cache, q, _wide_table(s), s.lengths, shared, groups, sm_scale=1.0), q, s, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("times,scale", [(1, 30.0), (1, 1e3), (1, 1e6), (1, 1e7), (1, 1e9), (1, 1e20), (1, 1e29), (2.0 ** 9, 1.0), (2.0 ** 9, 1e6)])
@pytest.mark.parametrize("batch,hq,hkv,d", [(40, 8, 2, 128), (40, 8, 2, 64), (2, 8, 2, 128)])
def test_scores_far_apart(batch, hq, hkv, d, times, scale, dtype):
    """Products of whole numbers, which float32 has exactly, with scales that leave no probability between 0 and those of the largest scores (e^-30 is below 2^-40): the output is the mean of
    these keys' values, off by its own rounding, and by 2^-24 of what was added up for each sum, weight and quotient."""
    s, shared, groups = _shared_setup([70], [batch], [1, 30, 100], hkv, d, 16, dtype, 11)
    for t in (s.cache.keys, s.cache.values):
        t.copy_(torch.randint(-4, 5, t.shape, generator=s.g, device="cuda"))
    s.cache.keys.mul_(times)
    q = (times * torch.randint(-4, 5, (batch, hq, d), generator=s.g, device="cuda")).to(dtype)
    out = _ops().paged_shared_decode_attention(s.cache, q, _wide_table(s), s.lengths, shared, groups, sm_scale=scale)
    u, group = torch.finfo(dtype).eps / 2, hq // hkv
    for b in range(batch):
        for h in range(hkv):
            got = out[b, h * group:(h + 1) * group].double()
            scores = q[b, h * group:(h + 1) * group].double() @ s.rows(s.cache.keys, b, h).T
            best, v = (scores == scores.amax(-1, keepdim=True)).double(), s.rows(s.cache.values, b, h)
            want = best @ v / best.sum(-1, keepdim=True)
            assert bool(((got - want).abs() <= 1.001 * u * want.abs() + 2.0 ** -20 * v.abs().max()).all()), (b, h)
    if scale > 30:  # (e^-30 is a number that can be the whole of an output, and sums have orders of their own)
        assert torch.equal(out, _ops().paged_decode_attention(s.cache, q, s.table, s.lengths, sm_scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefix,batch,hq,hkv,d,page", [(125, 128, 28, 4, 128, 64), (250, 32, 32, 8, 128, 128), (300, 100, 32, 8, 64, 64), (20, 9, 14, 2, 64, 16)])
def test_empty_groups_change_nothing(prefix, batch, hq, hkv, d, page, dtype):
    """A captured step has room for more groups than there are: the same bits as without it."""
    s, shared, groups = _shared_setup([prefix], [batch], [3, 70, 1], hkv, d, page, dtype, 5)
    table, q = _wide_table(s), s.queries(hq)
    want = _ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared)
    _close(want, q, s, d ** -0.5)
    for before, behind in ((0, 0), (0, 63), (1, 0), (70, 200)):
        pages, begins = _int32([5] * before + [prefix] + [9] * behind), _int32([0] * before + [0, batch] + [batch] * behind)
        assert torch.equal(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, pages, begins), want), (before, behind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefixes,sizes,hq,hkv,d", [
    ([200] + [3] * 40, [90] + [2] * 40, 32, 8, 64), ([2] * 70 + [100], [1] * 70 + [64], 32, 8, 128), ([100] * 3, [1] * 3, 28, 4, 128), ([400, 1, 400], [40, 1, 2], 28, 4, 128),
    ([50, 7] * 33, [1, 3] * 33, 14, 2, 64),
])
def test_groups_of_very_different_sizes(prefixes, sizes, hq, hkv, d, dtype):
    """A large group beside many small ones, and groups of one sequence, which share with nobody."""
    s, shared, groups = _shared_setup(prefixes, sizes, [40, 0, 1], hkv, d, 16, dtype, 6)
    table, q = _wide_table(s), s.queries(hq)
    _close(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups), q, s, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,hq,hkv,d,megabytes", [(16, 28, 4, 128, 272), (8, 32, 8, 128, 273), (6, 28, 4, 128, 335), (12, 14, 2, 64, 250), (1, 8, 2, 128, 1000), (1, 14, 2, 64, 500)])
def test_batches_that_the_caches_hold_are_plain_steps(batch, hq, hkv, d, megabytes):
    """The same bits as a plain step's, where room for all keys and values is below what makes sharing less time, or there is nobody to share with."""
    s, shared, groups = _shared_setup([40], [batch], [30, 1], hkv, d, 64, BF16, 3)
    pages = min(megabytes * 10 ** 6 // (batch * 64 * hkv * d * 4), (1 << 20) // 64)
    table = torch.cat([s.table, torch.zeros(batch, pages - s.table.shape[1], dtype=torch.int32, device="cuda")], 1)
    q = s.queries(hq)
    want = _ops().paged_decode_attention(s.cache, q, table, s.lengths)
    _close(want, q, s, d ** -0.5)
    assert torch.equal(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups), want)


def test_scratch_of_what_is_not_shared():
    """Parts of 256 work-groups, 35 MB with heads of 128, are there for the tables that may be shared only."""
    from anchor_attn.src.ops import _hip
    scratch = _hip.lib().aa_paged_shared_workspace_bytes
    assert scratch(2, 8, 2, 128, 16, 8, 1) < 1 << 20 and scratch(1, 8, 2, 128, 16, 65536, 1) < 10 << 20 and scratch(8, 32, 8, 128, 64, 128, 3) < 10 << 20
    assert scratch(12, 32, 8, 128, 64, 130, 3) > 30 << 20 and scratch(64, 14, 2, 64, 16, 1 << 12, 1) > 15 << 20


_SHARED = next(m for m in conversations.test_shared_decode.pytestmark if m.args[0].startswith("prefixes"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize(*_SHARED.args)
def test_shared_decode_in_wide_tables(prefixes, sizes, own, hq, hkv, d, page, layout, extra, alone, dtype):
    s, shared, groups = _shared_setup(prefixes, sizes, own, hkv, d, page, dtype, hq + page + 1, layout, extra, alone)
    conversations._check_shared_decode(s, _wide_table(s), shared, groups, s.queries(hq), len(sizes) == 1 and not alone)


@pytest.mark.gpu
@pytest.mark.parametrize("prefixes,sizes,hq,hkv,d,page", [([60, 9], [40, 3], 32, 8, 128, 64), ([300, 0, 40], [3, 1, 2], 14, 2, 64, 16)])
def test_captured_steps_on_two_streams(prefixes, sizes, hq, hkv, d, page):
    """Two captured steps whose groups, pages and lengths change between the replays, on a stream each and at once: the bits of eager steps."""
    ops, sets = _ops(), []
    for seed in range(2):
        s, shared, groups = _shared_setup(prefixes, sizes, [40, 0, 700], hkv, d, page, BF16, seed)
        s.cache.keys.nan_to_num_(0.5), s.cache.values.nan_to_num_(0.5)
        table, q, stream = _wide_table(s), s.queries(hq), torch.cuda.Stream()
        wants = []
        for pages, begins, fewer in ((shared, groups, 0), (shared // 2, groups, 3), (shared, torch.zeros_like(groups), 7), (shared * 0, groups, 0), (shared, groups, 100000)):
            lengths = (s.lengths - fewer).clamp(min=0)
            wants.append((pages.clone(), begins.clone(), lengths, ops.paged_shared_decode_attention(s.cache, q, table, lengths, pages, begins)))
        pages, begins, lengths = shared.clone(), groups.clone(), s.lengths.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            ops.paged_shared_decode_attention(s.cache, q, table, lengths, pages, begins)
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                out = ops.paged_shared_decode_attention(s.cache, q, table, lengths, pages, begins)
        torch.cuda.synchronize()
        # (a graph holds no reference to what it reads: the cache, the table and the queries live as long)
        sets.append((graph, stream, out, (pages, begins, lengths), wants, (s, table, q)))
    for i in [0, 1, 2, 3, 4, 0, 2, 1]:
        for graph, stream, _, given, wants, _ in sets:
            with torch.cuda.stream(stream):
                for x, y in zip(given, wants[i]):
                    x.copy_(y)
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, _, wants, _ in sets:
            assert torch.equal(out, wants[i][3]), i


@pytest.mark.gpu
def test_thousands_of_sequences_in_tables_for_a_million_keys():
    """Places that count more tiles than 32 bits have: the bits of a table for half as many keys."""
    batch, hq, hkv, d, page = 4096, 16, 8, 64, 256
    s, shared, groups = _shared_setup([5, 0, 2], [3000, 96, 1000], [3, 0, 40], hkv, d, page, BF16, 2)
    q, results = s.queries(hq), []
    for keys in (1 << 19, 1 << 20):
        table = torch.zeros(batch, keys // page, dtype=torch.int32, device="cuda")
        table[:, :s.table.shape[1]] = s.table
        results.append(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups))
    assert torch.equal(*results)
    plain = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    assert bool(((plain.float() - results[0].float()).abs() <= 2 ** -7 * plain.float().abs() + 2 ** -12).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("batch,hq,hkv,d,pages", [(40, 8, 2, 128, 70), (40, 8, 2, 64, 71), (3, 8, 2, 128, 33), (90, 28, 4, 128, 9)])
def test_infinite_values_of_shared_keys(batch, hq, hkv, d, pages, dtype):
    """Keys far below the largest (some 50 nats, where float32 has their probabilities) whose values are infinite or NaN: these channels are what 64 bits give, and the others are as close as ever."""
    s, shared, groups = _shared_setup([pages], [batch], [20, 0], hkv, d, 16, dtype, 13)
    s.cache.keys.mul_(0.3)
    s.cache.keys[s.table[0, 2].long(), :, 5] *= 2.0
    q = s.queries(hq, 1.0)
    q[:, :, 0] = 6.0
    s.cache.keys[s.table[0, 1].long(), :, :, 0] = -6.0
    for slot, channel, value in ((1, 3, float("inf")), (7, 4, float("-inf")), (9, 5, float("nan")), (2, 6, float("inf")), (3, 6, float("-inf"))):
        s.cache.values[s.table[0, 1].long(), 0, slot, channel] = value
    out = _ops().paged_shared_decode_attention(s.cache, q, _wide_table(s), s.lengths, shared, groups, sm_scale=1.0)
    u, group = torch.finfo(dtype).eps / 2, hq // hkv
    for b in range(batch):
        for h in range(hkv):
            got, x = out[b, h * group:(h + 1) * group].double(), q[b, h * group:(h + 1) * group].double()
            k, v = s.rows(s.cache.keys, b, h), s.rows(s.cache.values, b, h)
            p = (x @ k.T).softmax(-1)
            bad = ~v.isfinite().all(0)
            assert int(bad.sum()) == (4 if h == 0 else 0) and bool((p[:, 16:32] > 2.0 ** -100).all())
            if h == 0:
                assert bool((got[:, 3] == float("inf")).all()) and bool((got[:, 4] == float("-inf")).all()) and bool(got[:, 5:7].isnan().all())
            v = v.nan_to_num(0.0, 0.0, 0.0)
            want, magnitude = p @ v, (x.abs() @ k.abs().T).amax(-1, keepdim=True)
            bound = 1.001 * u * want.abs() + (2.0 * d * 2.0 ** -24 * magnitude + 2.0 ** -14 + u * u + k.shape[0] * 2.0 ** -24) * (p @ v.abs()) + 2.0 ** -25
            assert bool(((got - want).abs() <= bound)[:, ~bad].all()), (b, h, float(((got - want).abs() - bound)[:, ~bad].max()))
