"""Steps that count attention, where units are cut between work-groups and their parts joined."""
import pytest
import torch

from test_paged_cache import BF16, F16, _ops, _Setup
from test_paged_conversations import _weights_close, _weights_of


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,d", [(1700, 64), (2000, 128), (5000, 64)])
def test_parts_whose_scores_are_all_nan(n, d, dtype):
    """The keys of a KV head are NaN from some tile on, for each tile, so that parts of its unit have no other keys: its heads' outputs and all of its counted weights are NaN, and no others."""
    s = _Setup([n, n - 100], 2, d, 16, dtype, n, extra=200)
    s.cache = _weights_of(s)
    q, keys, before = s.queries(8), s.cache.keys.clone(), s.cache.weights.clone()
    at = s.table[0, :(n + 15) // 16].long()
    want = _ops().paged_weighing_decode_attention(s.cache, q, s.table, s.lengths, n_first=33)
    counted = s.cache.weights.clone()
    _weights_close(counted, before, q, s, d ** -0.5, 33)
    for tile in range(1, (n + 31) // 32):
        s.cache.keys.copy_(keys)
        s.cache.weights.copy_(before)
        s.cache.keys[at[2 * tile:], 0] = float("nan")
        out = _ops().paged_weighing_decode_attention(s.cache, q, s.table, s.lengths, n_first=33)
        assert bool(out[0, :4].isnan().all()) and torch.equal(out[0, 4:], want[0, 4:]) and torch.equal(out[1], want[1]), tile
        assert bool(s.cache.weights[at, 0].reshape(-1)[33:n].isnan().all()) and int(s.cache.weights.isnan().sum()) == n - 33, tile
        s.cache.weights[at, 0] = counted[at, 0]
        assert torch.equal(s.cache.weights, counted), tile


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hq,hkv,d", [([20001, 5], 71, 1, 64), ([3000, 9000, 0], 40, 2, 128), ([2500], 17, 1, 128)])
def test_groups_of_more_heads_than_a_unit_where_units_are_cut(lengths, hq, hkv, d, dtype):
    """Each block of 16 heads of a KV head has parts of its own, in groups that no power of two divides."""
    s = _Setup(lengths, hkv, d, 32, dtype, hq, extra=3)
    s.cache = _weights_of(s)
    s.cache.weights.uniform_(0, 2, generator=s.g)
    q, before = s.queries(hq), s.cache.weights.clone()
    out = _ops().paged_weighing_decode_attention(s.cache, q, s.table, s.lengths, n_first=100)
    assert torch.equal(out, _ops().paged_decode_attention(s.cache, q, s.table, s.lengths))
    _weights_close(s.cache.weights, before, q, s, d ** -0.5, 100)
