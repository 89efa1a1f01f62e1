"""Long and shared conversations in a key/value cache in pages - appending with norms and positions apart from places, decode that counts attention, eviction,
decode over a shared prefix - against plain float64 implementations, at the lengths, pages and layouts where tiles, pages and shares of the work end.

Tolerances beside those of tests/test_paged_cache.py (u: half a step of the 16-bit type).
Norm and rotation: a float32 sum of D squares is off by at most D * 2^-24 of it, its inverse root by half of that and 2^-22, three products by 2^-24 each,
the rotation by 2^-23 of its products' magnitudes: (D / 2 + 16) * 2^-24 of the magnitudes, and u of the result.
Weights: a probability is off by what tests/test_paged_cache.py says of it, 2 * D * 2^-24 * sum |q_d k_d| * scale + 2^-14 of it, a sum over the group's heads in float32 and the addition to
what was there by 2^-24 of each partial sum.
Over a prefix that more than 32 rows share (a group's queries of a KV head's group, on average) probabilities p_i are rounded once, by u of each at most, and their sum l is
that of the rounded ones: an output o = sum p_i v_i / l is off by sum d_i p_i (v_i - o) / l with |d_i| <= u, at most u (sum p_i |v_i| / l + |o|), 1 % more with
what is of second order."""

import ctypes
import pathlib

import pytest
import torch

from test_paged_cache import BF16, CACHE, EVERY, F16, READ, STEP, TOKENS, U, _close, _ops, _rotated, _Setup, _tables


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _weights_of(s):
    """A cache over the same tensors that keeps weights, 5.0 each at first."""
    keys = s.cache.keys
    return _ops().PagedCache(keys, s.cache.values, s.cache.bounds, torch.full(keys.shape[:3], 5.0, device="cuda"))


# ---- appending with norms, positions, rotated keys and weights -------------------------------------------------------

def _normed(x, weight, eps):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def _near(got, x, weight, eps, cos, sin):
    y = _normed(x, weight, eps)
    want, magnitude = _rotated(y, cos, sin)
    bound = U[got.dtype] * want.abs() * 1.001 + (x.shape[-1] / 2 + 16) * 2.0 ** -24 * magnitude + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("before,new,gone,hq,hkv,d,page,layout,padding", [
    ([0], [1], [0], 32, 8, 128, 64, "heads", 0),
    ([0, 63, 64, 17], [130, 1, 64, 0], [0, 5, 1000, 3], 28, 4, 128, 64, "rows", 5),
    ([5, 0, 31, 100], [1, 33, 2, 300], [700, 0, 1, 0], 14, 2, 64, 16, "heads", 0),
    ([0, 1, 255, 256], [257, 600, 1, 255], [0, 0, 9, 2], 8, 8, 128, 256, "part", 0),
    ([7] * 90, [1] * 90, list(range(90)), 4, 2, 64, 32, "heads", None),
    ([300] * 3, [517, 1, 90], [1, 2, 3], 71, 1, 64, 128, "part", 1),
])
def test_append_with_norms(before, new, gone, hq, hkv, d, page, layout, padding, dtype):
    """``padding`` None: a decode step, without starts."""
    ops = _ops()
    steps, padding, n, eps = padding is None, padding or 0, sum(new), 1e-3
    s = _Setup(before, hkv, d, page, dtype, len(before), layout, room=max(new))
    cache = _weights_of(s)
    scale = 10.0 ** torch.empty(n + padding, hq + 2 * hkv, 1, device="cuda").uniform_(-2, 1, generator=s.g)
    q, k, v = (torch.randn(n + padding, hq + 2 * hkv, d, generator=s.g, device="cuda") * scale).to(dtype).split((hq, hkv, hkv), 1)
    q[n // 2, 0] = 0.0  # (0 / sqrt(eps))
    wq, wk = ((1 + torch.randn(d, generator=s.g, device="cuda")).to(dtype) for _ in range(2))
    lengths = [a + b for a, b in zip(before, new)]
    had = [a + b for a, b in zip(lengths, gone)]
    cos, sin = _tables(max(had), d)
    starts = None if steps else _int32([sum(new[:b]) for b in range(len(new) + 1)])
    out, k_out = torch.full((n + padding, hq, d), 7.0, dtype=dtype, device="cuda"), torch.full((n + padding, hkv, d), 7.0, dtype=dtype, device="cuda")
    got = ops.append_to_pages(cache, q, k, v, cos, sin, s.table, _int32(lengths), starts, out, q_norm=wq, k_norm=wk, norm_eps=eps, positions=_int32(had), k_out=k_out)
    assert got is out and bool((out[n:] == 7.0).all()) and bool((k_out[n:] == 7.0).all())
    place = torch.tensor([p for a, b in zip(before, new) for p in range(a, a + b)], device="cuda")
    sequence = torch.tensor([i for i, b in enumerate(new) for _ in range(b)], device="cuda")
    position = place + torch.tensor(gone, device="cuda")[sequence]
    _near(out[:n], q[:n], wq, eps, cos[position], sin[position])
    _near(k_out[:n], k[:n], wk, eps, cos[position], sin[position])
    at, slot = s.table[sequence, place // page].long(), place % page
    assert torch.equal(cache.keys[at, :, slot], k_out[:n]) and torch.equal(cache.values[at, :, slot], v[:n])
    weights = torch.full_like(cache.weights, 5.0)
    weights[at, :, slot] = 0.0
    assert torch.equal(weights, cache.weights)
    for b, (a, c) in enumerate(zip(before, new)):
        for i in range(a // page, (a + c + page - 1) // page if c else 0):
            rows = cache.keys[int(s.table[b, i]), :, :min(page, a + c - i * page)]
            assert torch.equal(cache.bounds[int(s.table[b, i])], torch.stack((rows.amin(1), rows.amax(1)), 1))
    # in place, keys without queries, and without what is optional
    kept = cache.keys.clone()
    same = {"q_norm": wq, "k_norm": wk, "norm_eps": eps, "positions": _int32(had)}
    if n:
        mine_q, mine_k = q.clone(), k.clone()
        ops.append_to_pages(cache, mine_q, mine_k, v, cos, sin, s.table, _int32(lengths), starts, mine_q, k_out=mine_k, **same)
        assert torch.equal(mine_q[:n], out[:n]) and torch.equal(mine_k[:n], k_out[:n]) and torch.equal(mine_q[n:], q[n:]) and torch.equal(mine_k[n:], k[n:])
        mine_k = torch.zeros_like(k_out)
        assert ops.append_to_pages(s.cache, None, k, v, cos, sin, s.table, _int32(lengths), starts, k_out=mine_k, **{**same, "q_norm": None}) is None
        assert torch.equal(mine_k[:n], k_out[:n]) and torch.equal(cache.keys.nan_to_num(9.0), kept.nan_to_num(9.0))
        plain = ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table, _int32(lengths), starts)
        other = ops.append_to_pages(cache, q, k, v, cos, sin, s.table, _int32(lengths), starts, positions=_int32(lengths), k_out=mine_k)
        assert torch.equal(plain[:n], other[:n])  # (rows behind the last sequence are undefined)
        assert torch.equal(mine_k[:n], cache.keys[at, :, slot])


@pytest.mark.gpu
def test_a_cache_with_weights_is_copied_and_appended_to_without_angles():
    """Copies have weights of their own; keys that are rotated already set theirs to 0 and nobody else's; what the cache holds is what was given."""
    import copy
    s = _Setup([20, 0, 33], 2, 64, 16, BF16, 31)
    s.cache = _weights_of(s)
    s.cache.weights.fill_(3.0)
    other = copy.deepcopy(s.cache)
    assert torch.equal(other.weights, s.cache.weights) and other.weights.data_ptr() != s.cache.weights.data_ptr()
    k, v = (torch.randn(7, 2, 64, device="cuda").to(BF16) for _ in range(2))
    _ops().append_to_pages(other, None, k, v, None, None, s.table, s.lengths, _int32([0, 4, 4, 7]))
    new = [(0, 16 + i, i) for i in range(4)] + [(2, 30 + i, 4 + i) for i in range(3)]
    want = torch.full_like(other.weights, 3.0)
    for b, place, t in new:
        page = int(s.table[b, place // 16])
        want[page, :, place % 16] = 0.0
        assert torch.equal(other.keys[page, :, place % 16], k[t]) and torch.equal(other.values[page, :, place % 16], v[t])
    assert torch.equal(other.weights, want) and bool((s.cache.weights == 3.0).all())


@pytest.mark.gpu
def test_positions_that_angles_do_not_reach():
    """Tokens behind the angles are left out, and all of a sequence that has had fewer positions than it has keys."""
    ops = _ops()
    s = _Setup([0] * 4, 2, 64, 16, BF16, 5, room=40)
    cache = _weights_of(s)
    q, k, v = (torch.randn(20, h, 64, generator=s.g, device="cuda").to(BF16) for h in (4, 2, 2))
    cos, sin = _tables(100, 64)
    starts, lengths = _int32([0, 5, 10, 15, 20]), _int32([5, 5, 5, 5])
    out, k_out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    ops.append_to_pages(cache, q, k, v, cos, sin, s.table, lengths, starts, out, positions=_int32([4, 5, 102, 2 ** 31 - 1]), k_out=k_out)
    there = [5, 6, 7, 8, 9, 10, 11, 12]
    assert [i for i in range(20) if bool((out[i] != 7.0).any())] == there == [i for i in range(20) if bool((k_out[i] != 7.0).any())]
    assert int((cache.weights == 0).sum()) == 2 * len(there) and int((~cache.keys.isnan()).sum()) == len(there) * 2 * 64
    turned = cos[[0, 1, 2, 3, 4, 97, 98, 99]], sin[[0, 1, 2, 3, 4, 97, 98, 99]]
    want, magnitude = _rotated(q[there], *turned)
    assert bool(((out[there].double() - want).abs() <= U[BF16] * want.abs() * 1.001 + 2.0 ** -23 * magnitude + 2.0 ** -25).all())
    steps = {"positions": _int32([-(2 ** 31)] * 4)}
    before = cache.keys.clone()
    ops.append_to_pages(cache, q[:4], k[:4], v[:4], cos, sin, s.table, _int32([1, 2 ** 31 - 1, -(2 ** 31), 0]), **steps)
    assert torch.equal(cache.keys.nan_to_num(9.0), before.nan_to_num(9.0))


MORE = {"q_norm": 4096, "k_norm": 4096, "k_out": 4096, "ko_st": 256, "ko_sh": 128, "positions": 4096, "weights": 4096, "norm_eps": 1e-6}


@pytest.mark.parametrize("change,message", [
    *[(c, m) for c, m in EVERY if "given" not in c], ({"more": None}, "more is NULL"), ({"given": None}, "tokens is NULL"), ({"q_norm": 0}, "come together"), ({"k_norm": 0}, "come together"),
    ({"q": 0, "q_out": 0, "n_q_heads": 0}, "come together"), ({"cos": 0, "sin": 0}, "need cos and sin"), ({"q_norm": 4100}, "q_norm must be 16-byte"), ({"k_norm": 8}, "k_norm must be 16-byte"),
    ({"k_out": 8}, "k_out must be 16-byte"), ({"ko_sh": 4}, "k_out must have strides"), ({"positions": 6}, "positions must be 4-byte"), ({"weights": 5}, "weights must be 4-byte"),
    ({"norm_eps": -1e-6}, "norm_eps"), ({"norm_eps": float("nan")}, "norm_eps"), ({"norm_eps": 2.0}, "norm_eps"),
])
def test_what_the_c_interface_of_more_refuses(change, message):
    """Before anything is launched: the addresses are never read."""
    from anchor_attn.src.ops import _hip
    struct = _hip.PagedCacheStruct(*{**CACHE, **{k: v for k, v in change.items() if k in CACHE}}.values())
    packed = [None if name in change else pack.pack(*{**given, **{k: v for k, v in change.items() if k in given}}.values())
              for name, given, pack in (("given", TOKENS, _hip.PAGED_TOKENS), ("more", MORE, _hip.PAGED_MORE))]
    with pytest.raises(_hip.AnchorAttnHipError, match=message):
        _hip.check(_hip.lib().aa_paged_append_more(None if "cache" in change else ctypes.addressof(struct), *packed, None))


def _sizes_in_c(tmp_path, *expressions):
    import subprocess
    source = tmp_path / "sizes.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "anchor_attn_hip.h"\nint main(void) {\n'
                      + "".join(f'  printf("%zu ", (size_t)({x}));\n' for x in expressions) + "  return 0;\n}\n")
    include = pathlib.Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", f"-I{include}", "-o", tmp_path / "sizes", source], check=True)
    return [int(x) for x in subprocess.run([tmp_path / "sizes"], check=True, capture_output=True, text=True).stdout.split()]


def test_packed_more_is_laid_out_as_in_c(tmp_path):
    from anchor_attn.src.ops import _hip
    size, at = _sizes_in_c(tmp_path, "sizeof(aa_paged_more)", "offsetof(aa_paged_more, norm_eps)")
    assert size == _hip.PAGED_MORE.size and _hip.PAGED_MORE.pack(*[0] * 7, 1.0)[at:][:4] == b"\0\0\x80?"


@pytest.mark.gpu
def test_what_appending_refuses_beside():
    from anchor_attn.src.ops import _hip
    ops = _ops()
    z = lambda *shape, dtype=BF16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    keys, values, bounds = z(5, 2, 16, 64), z(5, 2, 16, 64), z(5, 2, 2, 64)
    wide = z(5, 2, 2, 16, 64)
    for weights in (z(5, 2, 16), z(5, 2, 17, dtype=torch.float32), z(5, 16, 2, dtype=torch.float32).transpose(1, 2), z(5, 2, 16, dtype=torch.float32).cpu(), z(5, 2, 16, dtype=torch.float32).requires_grad_(),
                    z(1000, dtype=torch.float32)[1:161].view(5, 2, 16), keys.view(-1)[:320].view(torch.float32).view(5, 2, 16), 1.0):
        with pytest.raises(_hip.AnchorAttnHipError):
            ops.PagedCache(keys, values, bounds, weights)
    with pytest.raises(_hip.AnchorAttnHipError):
        ops.PagedCache(wide[:, :, 0], wide[:, :, 1], None, wide.view(-1)[64:384].view(torch.float32).view(5, 2, 16))
    cache = ops.PagedCache(keys, values, bounds, z(5, 2, 16, dtype=torch.float32))
    assert ops.PagedCache.empty(5, 2, 16, 64, weights=True).weights.shape == (5, 2, 16) and ops.PagedCache.empty(5, 2, 16, 64).weights is None
    table, lengths, starts, cos = z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), z(3, dtype=torch.int32), z(50, 32, dtype=torch.float32)
    q, k, w = z(2, 4, 64), z(2, 2, 64), z(64)
    good = {"cache": cache, "q": q, "k": k, "v": k, "cos": cos, "sin": cos, "page_table": table, "lengths": lengths, "starts": starts, "q_norm": w, "k_norm": w, "positions": lengths, "k_out": z(2, 2, 64)}
    ops.append_to_pages(**good)
    for change in ({"q_norm": None}, {"k_norm": None}, {"q": None}, {"q": None, "cos": None, "sin": None}, {"q_norm": z(128)}, {"k_norm": z(64, dtype=F16)}, {"k_norm": w.cpu()}, {"q_norm": z(128)[::2]},
                   {"q_norm": z(72)[1:65]}, {"k_norm": [1.0] * 64}, {"norm_eps": -1.0}, {"norm_eps": float("nan")}, {"norm_eps": "x"}, {"positions": lengths.long()}, {"positions": z(3, dtype=torch.int32)},
                   {"positions": z(4, dtype=torch.int32)[::2]}, {"k_out": z(2, 4, 64)}, {"k_out": z(3, 2, 64)}, {"k_out": z(2, 1, 64).expand(2, 2, 64)}, {"k_out": z(2, 2, 64, dtype=F16)},
                   {"q_norm": z(64).requires_grad_()}, {"k_out": z(2, 2, 64).requires_grad_()}):
        with pytest.raises(_hip.AnchorAttnHipError):
            ops.append_to_pages(**{**good, **change})
    with pytest.raises(_hip.AnchorAttnHipError, match="need cos and sin"):
        ops.append_to_pages(cache, None, k, k, None, None, table, lengths, starts, positions=lengths)
    cache.weights.data = z(5, 2, 16, dtype=torch.float32)
    with pytest.raises(_hip.AnchorAttnHipError, match="other memory"):
        ops.append_to_pages(**good)
    torch.cuda.synchronize()


# ---- decode that counts attention ------------------------------------------------------------------------------------

LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 500, 1023]


def _weights_close(got, before, q, s, scale, n_first=0):
    """The weights of a cache after a step, all of them: what no sequence has a key for is as it was."""
    want, bound = before.double(), torch.zeros_like(before, dtype=torch.float64)
    group, page = q.shape[1] // s.hkv, s.page
    for b, n in enumerate(s.host):
        if n == 0:
            continue
        at = s.table[b, :(n + page - 1) // page].long()
        for h in range(s.hkv):
            x, k = q[b, h * group:(h + 1) * group].double(), s.rows(s.cache.keys, b, h)
            p = (x @ k.T * scale).softmax(-1)
            relative = 2.0 * s.d * 2.0 ** -24 * (x.abs() @ k.abs().T).amax(-1, keepdim=True) * scale + 2.0 ** -14 + n * 2.0 ** -24
            for t, add in ((want, p.sum(0)), (bound, (relative * p).sum(0) + (group + 1) * 2.0 ** -24 * p.sum(0))):
                rows = t[at, h].reshape(-1)
                rows[n_first:n] += add[n_first:]
                t[at, h] = rows.view(-1, page)
    err = (got.double() - want).abs()
    assert bool((err <= bound + torch.where(bound > 0, 2.0 ** -24 * want.abs(), 0.0)).all()), float((err - bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hq,hkv,d,page,layout,extra", [
    (LENGTHS, 32, 8, 128, 64, "heads", 0), (LENGTHS, 28, 4, 128, 16, "rows", 3), (LENGTHS, 14, 2, 64, 16, "heads", 100), (LENGTHS, 32, 8, 64, 32, "part", 0),
    (LENGTHS, 3, 3, 128, 256, "heads", 1), ([700, 1, 33], 17, 1, 128, 128, "rows", 0), ([900, 0], 71, 1, 64, 64, "heads", 0), ([20001], 32, 8, 128, 64, "heads", 0),
    ([9000, 40, 12345], 28, 4, 64, 16, "heads", 1), ([5], 14, 2, 64, 16, "heads", 0), ([0], 4, 2, 128, 16, "heads", 0), ([700] * 130 + [5000], 8, 2, 64, 64, "heads", 0),
    ([1] * 300, 14, 2, 64, 16, "heads", 0), ([16], 4, 2, 64, 16, "heads", 0),
])
def test_weighing_decode(lengths, hq, hkv, d, page, layout, extra, dtype):
    s = _Setup(lengths, hkv, d, page, dtype, hq + page, layout, extra=extra)
    cache, q = _weights_of(s), s.queries(hq)
    cache.weights.uniform_(0, 3, generator=s.g)
    before = cache.weights.clone()
    want = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    out = _ops().paged_weighing_decode_attention(cache, q, s.table, s.lengths)
    assert torch.equal(out, want)  # the same bits
    _weights_close(cache.weights, before, q, s, d ** -0.5)
    after = cache.weights.clone()
    cache.weights.copy_(before)
    assert _ops().paged_weighing_decode_attention(cache, q, s.table, s.lengths, out=torch.empty_like(q)).equal(want) and torch.equal(cache.weights, after)
    cache.weights.copy_(before)
    _ops().paged_weighing_decode_attention(cache, q, s.table, s.lengths, n_first=17, sm_scale=0.02)
    _weights_close(cache.weights, before, q, s, 0.02, 17)


@pytest.mark.gpu
@pytest.mark.parametrize("n_first", [1, 3, 4, 15, 33, 1023, 1025, 4999, 5000, 5001, 2 ** 31 - 1])
@pytest.mark.parametrize("lengths", [[5000], [700, 5000, 0, 3]])
def test_weighing_from_some_key_on(lengths, n_first):
    """Keys before n_first and rows behind the last key keep their weights; one short table and one whose steps are cut and joined."""
    s = _Setup(lengths, 2, 64, 16, BF16, 9, extra=1)
    s.cache = _weights_of(s)
    q, before = s.queries(8), s.cache.weights.clone()
    out = _ops().paged_weighing_decode_attention(s.cache, q, s.table, s.lengths, n_first=n_first)
    _close(out, q, s, 0.125)
    _weights_close(s.cache.weights, before, q, s, 0.125, n_first)
    short = min(lengths[0], 700)
    s.host = [short] + [0] * (len(lengths) - 1)
    before = s.cache.weights.clone()
    out = _ops().paged_weighing_decode_attention(s.cache, q, s.table[:, :44], _int32(s.host), n_first=n_first)
    _close(out, q, s, 0.125)
    _weights_close(s.cache.weights, before, q, s, 0.125, n_first)


@pytest.mark.gpu
def test_pages_far_into_a_large_pool():
    """Pages whose keys lie more than 2^32 bytes into the pool: every operator, the same bits as of the same pages in a small one."""
    ops = _ops()
    s = _Setup([300, 170, 300], 8, 128, 64, BF16, 12, room=10)
    s.table[1, :2] = s.table[0, :2]
    s.table[s.table < 0] = 0
    s.cache = _weights_of(s)
    far = 34000 - s.cache.n_pages
    big = ops.PagedCache.empty(34000, 8, 64, 128, weights=True)
    assert big.keys[far:].data_ptr() - big.keys.data_ptr() > 1 << 32
    for a, b in ((big.keys, s.cache.keys), (big.values, s.cache.values), (big.bounds, s.cache.bounds), (big.weights, s.cache.weights)):
        a[far:] = b
    wq, wk = (1 + torch.randn(128, device="cuda") / 4).to(BF16), (1 + torch.randn(128, device="cuda") / 4).to(BF16)
    cos, sin = _tables(400, 128)
    q, k, v = (torch.randn(3, h, 128, device="cuda").to(BF16) for h in (32, 8, 8))
    results = []
    for cache, table in ((s.cache, s.table), (big, (s.table.long() + far).clamp(max=33999).int())):
        lengths, roomy = s.lengths + 1, _roomy(s)
        roomy[:, :table.shape[1]] = table
        rotated = ops.append_to_pages(cache, q, k, v, cos, sin, table, lengths, q_norm=wq, k_norm=wk, positions=lengths + 3)
        shared = ops.paged_shared_decode_attention(cache, rotated, roomy, lengths, _int32([2]), _int32([0, 2]))
        counted = ops.paged_weighing_decode_attention(cache, rotated, table, lengths, n_first=128)
        new, kept = ops.evict_from_pages(cache, table, lengths, 160, n_first=128, n_last=4)
        here = slice(far if cache is big else 0, None)
        results.append([rotated, shared, counted, new, kept, *(t[here].nan_to_num(9.0) for t in (cache.keys, cache.values, cache.bounds, cache.weights))])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_weighing_scores_that_are_infinite_or_nan():
    """A key of minus infinity has no weight, a sequence whose scores are all of it or one of which is NaN or plus infinity NaN where its heads are, and no other."""
    s = _Setup([700, 40, 40, 40, 300], 2, 64, 16, BF16, 9)
    cache, q = _weights_of(s), s.queries(4, 0.5)
    q[:, :, 0] = 1.0
    for b, value in ((0, float("-inf")), (1, float("nan")), (2, float("inf"))):
        s.cache.keys[s.table[b, 1].long(), 0, 3, 0] = value
    s.cache.keys[s.table[3, :3].long(), 0, :, 0] = float("-inf")
    before = cache.weights.clone()
    out = _ops().paged_weighing_decode_attention(cache, q, s.table, s.lengths)
    assert [[bool(out[b, 2 * h:2 * h + 2].isnan().all()) for h in range(2)] for b in range(5)] == [[False, False], [True, False], [True, False], [True, False], [False, False]]
    weights = [[cache.weights[s.table[b, :(n + 15) // 16].long(), h].reshape(-1)[:n] for h in range(2)] for b, n in enumerate(s.host)]
    assert all(bool(weights[b][0].isnan().all()) for b in (1, 2, 3)) and int(cache.weights.isnan().sum()) == 120
    assert float(weights[0][0][19]) == 5.0 and bool((weights[0][0][:19] > 5.0).all())
    # and infinite values have no part in it
    cache.weights.copy_(before)
    s.cache.values[s.table[4, 0].long(), 0, 5, 3] = float("inf")
    again = _ops().paged_weighing_decode_attention(cache, q, s.table, s.lengths)
    assert bool((again[4, :2, 3] == float("inf")).all()) and torch.equal(weights[4][0], cache.weights[s.table[4, :19].long(), 0].reshape(-1)[:300])


@pytest.mark.gpu
def test_weighing_of_lengths_and_pages_that_do_not_fit():
    """Lengths above the table are its size; a page outside the pool is read as the nearest one, and nothing is added for it."""
    s = _Setup([64, 64, 64], 2, 64, 16, BF16, 10)
    cache, q = _weights_of(s), s.queries(4)
    s.cache.keys.nan_to_num_(0.5), s.cache.values.nan_to_num_(0.5)
    s.table[1, 2], s.table[1, 3] = -5, 2 ** 31 - 1
    lengths = _int32([1000, 64, -3])
    out = _ops().paged_weighing_decode_attention(cache, q, s.table, lengths)
    assert torch.equal(out, _ops().paged_decode_attention(s.cache, q, s.table, lengths))
    at = torch.cat((s.table[0], s.table[1, :2])).long()
    changed = (cache.weights != 5.0).any(-1).any(-1)
    assert sorted(changed.nonzero().flatten().tolist()) == sorted(at.tolist())


# ---- decode over a shared prefix -----------------------------------------------------------------------------------

def _shared_setup(prefixes, sizes, own, hkv, d, page, dtype, seed, layout="heads", extra=0, alone=()):
    """Groups of ``sizes`` sequences with ``prefixes`` pages in common and ``own`` keys each, after the sequences ``alone`` of no group."""
    lengths = list(alone)
    group_of = [None] * len(alone)
    for g, n in enumerate(sizes):
        for _ in range(n):
            lengths.append(prefixes[g] * page + own[(len(lengths) - len(alone)) % len(own)])
            group_of.append(g)
    s = _Setup(lengths, hkv, d, page, dtype, seed, layout, extra=extra)
    begins = [len(alone)]
    for n in sizes:
        begins.append(begins[-1] + n)
    for b, g in enumerate(group_of):
        if g is not None:
            s.table[b, :prefixes[g]] = s.table[begins[g], :prefixes[g]]
    return s, _int32(prefixes), _int32(begins)


def _roomy(s):
    """The setup's table with room for so many pages (zeros, which nothing reads) that the kernels for shared pages are what runs, and that the caches do not hold them all."""
    pages = 300_000_000 // (s.table.shape[0] * s.cache.page_size * s.hkv * s.d * 4) + 1
    return torch.cat([s.table, torch.zeros(s.table.shape[0], max(pages - s.table.shape[1], 0), dtype=torch.int32, device="cuda")], 1)


def _shared_close(out, q, s, scale, n_groups):
    """What :func:`_close` asks for, and where more than 16 rows (32 with heads of 64) share a prefix the rounding of probabilities."""
    group = q.shape[1] // s.hkv
    if q.shape[0] * group // n_groups <= (32 if s.d == 64 else 16):
        return _close(out, q, s, scale)
    for b in range(q.shape[0]):
        for h in range(s.hkv):
            got = out[b, h * group:(h + 1) * group].double()
            if s.host[b] == 0:
                assert bool((got == 0).all())
                continue
            k, v, x = s.rows(s.cache.keys, b, h), s.rows(s.cache.values, b, h), q[b, h * group:(h + 1) * group].double()
            p = (x @ k.T * scale).softmax(-1)
            want = p @ v
            relative = 2.0 * s.d * 2.0 ** -24 * (x.abs() @ k.abs().T).amax(-1, keepdim=True) * scale + 2.0 ** -14 + k.shape[0] * 2.0 ** -24 + 1.01 * U[out.dtype]
            bound = 2.02 * U[out.dtype] * want.abs() + relative * (p @ v.abs()) + 2.0 ** -25
            err = (got - want).abs()
            assert bool((err <= bound).all()), (b, h, float((err - bound).max()), float(err.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefixes,sizes,own,hq,hkv,d,page,layout,extra,alone", [
    ([3], [5], [1, 40, 300], 32, 8, 128, 64, "heads", 0, []),
    ([1], [2], [1], 14, 2, 64, 16, "heads", 0, []),
    ([5], [1], [0], 4, 2, 128, 16, "heads", 0, []),
    ([7, 0, 33, 2], [6, 3, 17, 1], [3, 0, 130, 16], 28, 4, 128, 16, "rows", 2, [5, 0, 700]),
    ([40], [70], [17, 1, 0, 90], 28, 4, 128, 32, "part", 0, []),
    ([9, 13, 1], [40, 1, 30], [33, 64], 32, 8, 64, 256, "heads", 1, [1]),
    ([300], [9], [20], 71, 1, 64, 16, "heads", 0, []),
    ([157], [33], [7, 1000], 8, 2, 128, 64, "heads", 0, []),
    ([313], [3], [2], 8, 2, 128, 64, "rows", 0, [9000]),
    ([2] * 90, [3] * 90, [5, 1, 20], 4, 1, 64, 32, "heads", 0, [7] * 5),
    ([1, 4096], [1, 2], [33], 4, 2, 64, 16, "heads", 0, []),
    ([0, 0, 3], [2, 0, 2], [9], 4, 2, 64, 16, "heads", 0, []),
    ([3, 2, 5] * 40, [2, 0, 1] * 40, [9, 0], 4, 2, 64, 16, "heads", 0, [3]),
    ([70], [32], [20, 0, 3], 32, 8, 128, 64, "heads", 0, []),
    ([70], [33], [20, 0, 3], 32, 8, 128, 64, "heads", 0, [5]),
    ([1], [300], [1], 1, 1, 128, 256, "heads", 0, []),
])
def test_shared_decode(prefixes, sizes, own, hq, hkv, d, page, layout, extra, alone, dtype):
    s, shared, groups = _shared_setup(prefixes, sizes, own, hkv, d, page, dtype, hq + page, layout, extra, alone)
    for table in (_roomy(s), s.table):
        _check_shared_decode(s, table, shared, groups, s.queries(hq), len(sizes) == 1 and not alone)


def _check_shared_decode(s, table, shared, groups, q, all_in_one):
    hq, d, dtype, n_groups = q.shape[1], s.d, q.dtype, len(shared)
    wide = torch.full((len(s.host), hq + 1, d + 8), 7.0, dtype=dtype, device="cuda")
    out = wide[:, 1:, 8:]
    assert _ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups, out=out) is out
    assert bool((wide[:, 0] == 7.0).all()) and bool((wide[:, :, :8] == 7.0).all())
    _shared_close(out, q, s, d ** -0.5, n_groups)
    again = _ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups, sm_scale=d ** -0.5)
    assert torch.equal(out, again)  # the same bits
    _shared_close(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups, sm_scale=0.3), q, s, 0.3, n_groups)
    if all_in_one:
        assert torch.equal(_ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared), out)
    assert _ops().paged_shared_decode_attention(s.cache, q, table, s.lengths, shared, groups, out=q) is q and torch.equal(q, again)


@pytest.mark.gpu
def test_shared_decode_of_sequences_that_are_shorter_than_the_prefix():
    """A padded batch and sequences that do not have all of it: what they do not see, an infinite value too, does not reach them."""
    s, shared, groups = _shared_setup([10, 6], [8, 4], [40], 2, 64, 16, BF16, 3)
    s.host = [165, 0, 159, 160, 1, 200, 0, 161, 96, 95, 16, 97]
    s.lengths.copy_(_int32(s.host))
    s.cache.values.nan_to_num_(1.0), s.cache.keys.nan_to_num_(1.0)
    q = s.queries(8)
    got = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups)
    _close(got, q, s, 0.125)
    s.cache.values[s.table[0, 9].long(), :, 15] = float("inf")  # (key 159)
    s.cache.keys[s.table[8, 5].long(), :, 15] = float("nan")  # (key 95)
    bad = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups)
    seen = [b for b, n in enumerate(s.host) if n >= (160 if b < 8 else 96)]
    assert all(not bool(bad[b].isfinite().any()) if b in seen else torch.equal(bad[b], got[b]) for b in range(12))
    assert all(bool((bad[b] == float("inf")).all()) for b in seen if b < 8) and all(bool(bad[b].isnan().all()) for b in seen if b >= 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("batch,pages", [(3, 4), (40, 300)])
def test_shared_decode_with_infinite_values_and_scores(batch, pages, dtype):
    """In the prefix: an infinite value gives an infinity in its channel and nothing else; keys that are all minus infinity leave the own ones, and the other way round."""
    s, shared, groups = _shared_setup([pages], [batch], [40], 2, 64, 16, dtype, 8)
    q = s.queries(8, 0.3)
    q[:, :, 0] = 1.0
    want = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups)
    at = s.table[0, 1].long()
    s.cache.values[at, 0, 3, 5], s.cache.values[at, 0, 4, 6], s.cache.values[at, 0, 9, 7] = float("inf"), float("-inf"), float("nan")
    got = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups)
    assert bool((got[:, :4, 5] == float("inf")).all()) and bool((got[:, :4, 6] == float("-inf")).all()) and bool(got[:, :4, 7].isnan().all())
    assert torch.equal(got[:, 4:], want[:, 4:])
    rest = torch.ones(64, dtype=torch.bool, device="cuda")
    rest[5:8] = False
    # (probabilities rounded once may have been so relative to different maxima: values below 4 by 2 u each way)
    slack = 8 * U[dtype] if batch * 4 > 32 else 0.0
    assert bool(((got[:, :4, rest] - want[:, :4, rest]).abs() <= 2 * U[dtype] * want[:, :4, rest].abs() + 2.0 ** -13 + slack).all())
    # minus infinity: the keys of the prefix for KV head 0, all own keys of sequence 1 for KV head 1, all of sequence 2 for both
    s.cache.values[at, 0, :, 5:8] = 0.5
    s.cache.keys[s.table[0, :pages].long(), 0, :, 0] = float("-inf")
    s.cache.keys[s.table[1, pages:pages + 3].long(), 1, :, 0] = float("-inf")
    s.cache.keys[s.table[2, pages:pages + 3].long(), 0, :, 0] = float("-inf")
    got = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups)
    plain = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    assert bool(got[2, :4].isnan().all()) and bool(plain[2, :4].isnan().all()) and int(got.isnan().sum()) == 4 * 64
    near = (got.double() - plain.double()).abs() <= 2 * U[dtype] * plain.abs() + 2.0 ** -12 + slack
    assert bool((near | plain.isnan()).all())


@pytest.mark.gpu
def test_groups_that_do_not_fit():
    """Begins outside the batch, more pages than the table has, pages outside the pool: everything is clamped, and outside of groups all is as it was."""
    s, shared, groups = _shared_setup([4], [6], [20], 2, 64, 16, BF16, 4)
    s.cache.keys.nan_to_num_(0.5), s.cache.values.nan_to_num_(0.5)
    q = s.queries(4)
    plain = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    for shared_pages, begins in (([2 ** 31 - 1], [0, 6]), ([-5], [0, 6]), ([4], [-7, 2 ** 31 - 1]), ([4, 4], [-9, 2, 100]), ([4], [6, 6]), ([4], [5, 3]), ([4, 4, 4], [2, 2, 2, 4]), ([4], [-3, -1])):
        got = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, _int32(shared_pages), _int32(begins))
        assert bool(((got.float() - plain.float()).abs() <= 2 * U[BF16] * plain.float().abs() + 2.0 ** -12).all()), (shared_pages, begins)
    s.table[0, 1], s.table[0, 2] = -1, 2 ** 31 - 1
    got = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups)
    s.table[:, 1], s.table[:, 2] = 0, s.cache.n_pages - 1
    assert torch.equal(got, _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), s.lengths, shared, groups))
    # no keys but the prefix, in a table that ends with it
    s.host = [64] * 6
    got = _ops().paged_shared_decode_attention(s.cache, q, s.table[:, :4], _int32(s.host), shared, groups)
    _close(got, q, s, 0.125)
    got = _ops().paged_shared_decode_attention(s.cache, q, _roomy(s), _int32(s.host), shared, groups)
    _close(got, q, s, 0.125)


STEPS = {"weigh": ("aa_paged_weighing_decode_fwd", {"weights": 4096, "n_first": 0}), "shared": ("aa_paged_shared_decode_fwd", {"shared_pages": 4096, "groups": 4096, "n_groups": 2})}


@pytest.mark.parametrize("fn,change,message", [
    *[(fn, c, m) for fn in STEPS for c, m in EVERY + READ], *[(fn, {"workspace_bytes": 100}, "workspace has 100 bytes") for fn in STEPS], *[(fn, {"workspace": 0}, "workspace is NULL") for fn in STEPS],
    ("weigh", {"weights": 0}, "weights is NULL"), ("weigh", {"weights": 4100}, "weights must be 16-byte"), ("weigh", {"n_first": -1}, "n_first"),
    ("shared", {"shared_pages": 0}, "shared_pages is NULL"), ("shared", {"groups": 0}, "groups is NULL"), ("shared", {"groups": 6}, "groups must be 4-byte"), ("shared", {"shared_pages": 5}, "shared_pages must be 4-byte"),
    ("shared", {"n_groups": 0}, "0 groups"), ("shared", {"n_groups": 65536}, "65536 groups"),
])
def test_what_the_c_interface_of_steps_refuses(fn, change, message):
    """Before anything is launched: the addresses are never read."""
    from anchor_attn.src.ops import _hip
    name, more = STEPS[fn]
    assert set(change) <= {*STEP, *more, *CACHE, "cache", "given"}
    struct = _hip.PagedCacheStruct(*{**CACHE, **{k: v for k, v in change.items() if k in CACHE}}.values())
    step = _hip.PAGED_STEP.pack(*{**STEP, **{k: v for k, v in change.items() if k in STEP}}.values())
    with pytest.raises(_hip.AnchorAttnHipError, match=message):
        _hip.check(getattr(_hip.lib(), name)(None if "cache" in change else ctypes.addressof(struct), None if "given" in change else step,
                                             *{**more, **{k: v for k, v in change.items() if k in more}}.values(), None))


def test_scratch_of_steps():
    from anchor_attn.src.ops import _hip
    lib = _hip.lib()
    assert lib.aa_paged_weighing_workspace_bytes(0, 8, 2, 128, 16, 8) == 0 == lib.aa_paged_shared_workspace_bytes(2, 0, 2, 128, 16, 8, 1) == lib.aa_paged_shared_workspace_bytes(2, 8, 2, 128, 16, 8, 0)
    assert lib.aa_paged_weighing_workspace_bytes(2, 8, 2, 128, 16, 8) >= 2 * 8 * (16 * 8 + 2) * 4
    assert lib.aa_paged_weighing_workspace_bytes(128, 32, 8, 128, 16, 65536) >= 128 * 32 * (1 << 22)
    assert lib.aa_paged_shared_workspace_bytes(2, 8, 2, 128, 16, 8, 1) >= 2 * 8 * 130 * 4


@pytest.mark.gpu
def test_what_steps_refuse():
    from anchor_attn.src.ops import _hip
    ops = _ops()
    z = lambda *shape, dtype=BF16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    cache = ops.PagedCache.empty(5, 2, 16, 64, weights=True)
    for t in (cache.keys, cache.values, cache.weights):
        t.zero_()
    table, lengths, q = z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), z(2, 4, 64)
    good = {"cache": cache, "q": q, "page_table": table, "lengths": lengths}
    one = z(1, dtype=torch.int32)
    reads = [{"q": z(2, 3, 64)}, {"q": z(3, 4, 64)}, {"q": q.cpu()}, {"q": z(2, 4, 64).requires_grad_()}, {"page_table": table.long()}, {"lengths": lengths.long()}, {"out": z(2, 4, 128)},
             {"out": z(1, 4, 64).expand(2, 4, 64)}, {"sm_scale": 0.0}, {"sm_scale": float("nan")}, {"cache": None}]
    for fn, base, changes in ((ops.paged_weighing_decode_attention, good, reads + [{"n_first": -1}, {"n_first": 1.5}, {"n_first": None}, {"n_first": 1 << 31}, {"cache": ops.PagedCache(cache.keys, cache.values)}]),
                              (ops.paged_shared_decode_attention, {**good, "shared_pages": one, "groups": lengths},
                               reads + [{"shared_pages": one.long()}, {"shared_pages": z(2, dtype=torch.int32)}, {"shared_pages": one.cpu()}, {"shared_pages": None}, {"shared_pages": z(0, dtype=torch.int32), "groups": one},
                                        {"groups": one}, {"groups": z(4, dtype=torch.int32)[::2]}, {"shared_pages": z(2, dtype=torch.int32), "groups": None}, {"shared_pages": z(1, 1, dtype=torch.int32)}])):
        fn(**base)
        for change in changes:
            with pytest.raises(_hip.AnchorAttnHipError):
                fn(**{**base, **change})
        with pytest.raises(_hip.AnchorAttnHipError, match="traced"):
            torch.func.vmap(lambda x: fn(**{**base, "q": x}))(q[None])
        assert fn(**{**base, "q": q[:0], "page_table": table[:0], "lengths": lengths[:0]}).shape == (0, 4, 64)
    torch.cuda.synchronize()


# ---- giving up keys --------------------------------------------------------------------------------------------------

def _kept(weights, n, n_keys, n_first, n_last):
    """The places by their definition, of a sequence and KV head, sorted on the host."""
    w = [float("inf") if x != x else x for x in weights.tolist()]
    best = sorted(range(n_first, n - n_last), key=lambda i: (-w[i], i))[:n_keys - n_first - n_last]
    return [*range(n_first), *sorted(best), *range(n - n_last, n)]


def _evict_and_check(s, cache, n_keys, n_first, n_last, above=None):
    """All of the cache's tensors and what is returned, bit for bit."""
    page = s.page
    want = {x: getattr(cache, x).clone() for x in ("keys", "values", "bounds", "weights")}
    kept = torch.full((len(s.host), s.hkv, n_keys), -1, dtype=torch.int32)
    old = {x: t.clone() for x, t in want.items()}
    for b, n in enumerate(s.host):
        if n <= (n_keys if above is None else above):
            continue
        at = s.table[b, :(n + page - 1) // page].long()
        for h in range(s.hkv):
            mine = _kept(old["weights"][at, h].reshape(-1)[:n], n, n_keys, n_first, n_last)
            kept[b, h] = torch.tensor(mine, dtype=torch.int32)
            to = at[:(n_keys + page - 1) // page]
            for x in ("keys", "values", "weights"):
                rows = want[x][to, h].flatten(0, 1)
                rows[:n_keys] = old[x][at, h].flatten(0, 1)[torch.tensor(mine, device="cuda")]
                want[x][to, h] = rows.unflatten(0, (-1, page))
            changed = next((i for i, x in enumerate(mine) if x != i), n_keys)
            for i in range(changed // page, (n_keys + page - 1) // page):
                rows = want["keys"][to[i], h, :min(page, n_keys - i * page)]
                want["bounds"][to[i], h] = torch.stack((rows.amin(0), rows.amax(0)))
    lengths, got = _ops().evict_from_pages(cache, s.table, s.lengths, n_keys, n_first, n_last, above)
    assert got.dtype == lengths.dtype == torch.int32 and torch.equal(got.cpu(), kept)
    s.host = [n_keys if n > (n_keys if above is None else above) else n for n in s.host]
    assert lengths.tolist() == s.host
    for x, t in want.items():
        mine = getattr(cache, x)
        assert torch.equal(mine.isnan(), t.isnan()) and torch.equal(mine.nan_to_num(9.0), t.nan_to_num(9.0)), x
    return lengths


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hkv,d,page,layout,n_keys,n_first,n_last,above", [
    (LENGTHS, 8, 128, 64, "heads", 40, 4, 10, None), (LENGTHS, 4, 128, 16, "rows", 16, 0, 0, None), (LENGTHS, 2, 64, 16, "heads", 1, 0, 1, None), (LENGTHS, 2, 64, 32, "part", 33, 0, 1, 64),
    (LENGTHS, 3, 128, 256, "heads", 300, 17, 30, 301), ([700, 1, 33], 1, 128, 128, "rows", 33, 33, 0, None), ([900, 0], 1, 64, 64, "heads", 700, 100, 600, None),
    ([20001], 8, 128, 64, "heads", 4096, 4, 500, None), ([9000, 40, 12345], 4, 64, 16, "heads", 8999, 1, 2, None), ([5], 2, 64, 16, "heads", 5, 1, 1, None), ([0], 2, 128, 16, "heads", 3, 0, 0, None),
    ([130] * 70, 2, 64, 64, "heads", 128, 0, 64, None), ([17], 2, 64, 16, "heads", 1, 0, 0, None), ([70001], 1, 64, 16, "heads", 64000, 0, 1, None), ([1000, 2000], 2, 64, 16, "heads", 100000, 10, 10, None),
    ([1 << 17], 1, 64, 256, "heads", 1000, 1, 1, None), ([36864, 36865, 5000], 2, 64, 128, "heads", 3001, 5, 100, None), ([1100, 1500, 900] * 30, 2, 128, 16, "rows", 1000, 0, 500, None),
    ([5000, 4400, 3999], 2, 128, 32, "heads", 4000, 600, 900, 4001), ([300000], 1, 64, 64, "heads", 150000, 0, 0, None),
])
def test_evict(lengths, hkv, d, page, layout, n_keys, n_first, n_last, above, dtype):
    s = _Setup(lengths, hkv, d, page, dtype, hkv + page, layout, extra=1)
    cache = _weights_of(s)
    cache.weights.normal_(generator=s.g).mul_(3).exp_()
    got = _evict_and_check(s, cache, n_keys, n_first, n_last, above)
    # once more: nothing is left to give up, or the weights have moved along
    s.lengths = got
    _evict_and_check(s, cache, max(1, n_keys // 2), n_first // 2, n_last // 2)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [50, 3000])
def test_evict_by_weights_that_are_equal_nan_or_of_any_sign(n):
    """Equal weights go by place, -0 is 0, NaN is infinity, and negative ones are the smallest."""
    for seed, values in enumerate(([1.0], [0.0, -0.0, 1e-45], [float("nan"), float("inf"), 1.0, -float("nan")], [-1.0, -float("inf"), 0.0, 1e-38, 2.0], [1.0, 1.0 + 2.0 ** -23, 1.0 + 2.0 ** -22])):
        s = _Setup([n, n - 7], 2, 64, 16, F16, seed, extra=1)
        cache = _weights_of(s)
        cache.weights.copy_(torch.tensor(values, device="cuda")[torch.randint(len(values), cache.weights.shape, generator=s.g, device="cuda")])
        _evict_and_check(s, cache, n // 2, 3, 5)


@pytest.mark.gpu
def test_bounds_of_moved_keys_that_are_nan_or_infinite():
    s = _Setup([200], 2, 64, 16, F16, 6)
    cache = _weights_of(s)
    cache.weights.uniform_(generator=s.g)
    at = s.table[0].long()
    cache.keys[at[11], 0, 3, 5], cache.keys[at[10], 0, 2, 6], cache.keys[at[9], 1, 1, 7], cache.keys[at[8], 1, 1, 8] = float("nan"), float("inf"), float("-inf"), -float("nan")
    for i, h, r in ((11, 0, 3), (10, 0, 2), (9, 1, 1), (8, 1, 1)):
        cache.weights[at[i], h, r] = 2.0
    _evict_and_check(s, cache, 60, 1, 1)
    seen = torch.cat([cache.bounds[at[i], h].flatten() for i in range(4) for h in range(2)])
    assert int(seen.isnan().sum()) == 4 and int(seen.isinf().sum()) == 2


@pytest.mark.gpu
def test_evict_without_bounds_and_of_what_does_not_fit():
    """Lengths above the table are its size; a page outside the pool is read as the nearest one and not written."""
    s = _Setup([64, 64, 64, 64], 2, 64, 16, BF16, 10)
    keys, values = s.cache.keys.nan_to_num(0.5), s.cache.values.nan_to_num(0.5)
    cache = _ops().PagedCache(keys, values, None, torch.rand(keys.shape[:3], generator=s.g, device="cuda"))
    before = keys.clone(), values.clone(), cache.weights.clone()
    s.table[1, 0], s.table[2, 3] = -5, 2 ** 31 - 1
    lengths, kept = _ops().evict_from_pages(cache, s.table, _int32([1000, 64, 64, -3]), 20, 2, 3)
    assert lengths.tolist() == [20, 20, 20, 0] and bool((kept[3] == -1).all())
    for b, pages in ((0, s.table[0]), (1, torch.cat((_int32([0]), s.table[1, 1:]))), (2, torch.cat((s.table[2, :3], _int32([cache.n_pages - 1]))))):
        for h in range(2):
            mine = _kept(before[2][pages.long(), h].reshape(-1), 64, 20, 2, 3)
            assert kept[b, h].tolist() == mine
            for i, x in enumerate(mine):
                if b == 1 and i < 16:
                    continue  # (in a page outside the pool)
                for t, u in ((keys, before[0]), (values, before[1]), (cache.weights, before[2])):
                    assert torch.equal(t[int(pages[i // 16]), h, i % 16], u[int(pages[x // 16]), h, x % 16])
    written = {int(x) for x in torch.cat((s.table[0, :2], s.table[1, 1:2], s.table[2, :2]))}
    for t, u in zip((keys, values, cache.weights), before):
        assert all(torch.equal(t[i], u[i]) for i in range(cache.n_pages) if i not in written)


EVICTION = {"page_table": 4096, "pt_sb": 8, "lengths": 4096, "new_lengths": 8192, "kept": 4096, "weights": 4096, "workspace": 4096, "workspace_bytes": 1 << 40, "batch": 2, "max_pages": 100,
            "n_keys": 1000, "n_first": 2, "n_last": 3, "above": 1200}


@pytest.mark.parametrize("change,message", [
    *[(c, m) for c, m in EVERY if not {"q", "q_sh"} & set(c) and m != "must divide"], ({"weights": 0}, "weights is NULL"), ({"weights": 4100}, "weights must be 16-byte"),
    ({"new_lengths": 0}, "new_lengths is NULL"), ({"kept": 0}, "kept is NULL"), ({"kept": 6}, "kept must be 4-byte"), ({"workspace": 0}, "workspace is NULL"), ({"workspace_bytes": 100}, "workspace has 100 bytes"),
    ({"n_keys": 0}, "not supported"), ({"n_keys": 4}, "not supported"), ({"n_first": -1}, "not supported"), ({"n_last": -1}, "not supported"), ({"n_first": 998}, "not supported"),
    ({"n_first": 2 ** 31 - 1, "n_last": 2 ** 31 - 1}, "not supported"), ({"above": 999}, "not supported"), ({"n_keys": (1 << 20) + 1, "above": 1 << 21}, "not supported"),
    ({"batch": 65535, "n_kv_heads": 512, "kp_sh": 128}, "2\\^24"), ({"new_lengths": 4096}, "share memory"), ({"new_lengths": 4092}, "share memory"),
])
def test_what_the_c_interface_of_eviction_refuses(change, message):
    """Before anything is launched: the addresses are never read."""
    from anchor_attn.src.ops import _hip
    assert set(change) <= {*EVICTION, *CACHE, "cache", "given"}
    struct = _hip.PagedCacheStruct(*{**CACHE, **{k: v for k, v in change.items() if k in CACHE}}.values())
    with pytest.raises(_hip.AnchorAttnHipError, match=message):
        _hip.check(_hip.lib().aa_paged_evict(None if "cache" in change else ctypes.addressof(struct),
                                             None if "given" in change else _hip.PAGED_EVICTION.pack(*{**EVICTION, **{k: v for k, v in change.items() if k in EVICTION}}.values()), None))


def test_packed_eviction_is_laid_out_as_in_c(tmp_path):
    from anchor_attn.src.ops import _hip
    size, at = _sizes_in_c(tmp_path, "sizeof(aa_paged_eviction)", "offsetof(aa_paged_eviction, above)")
    assert size == _hip.PAGED_EVICTION.size and _hip.PAGED_EVICTION.pack(*range(14))[at] == 13
    assert _hip.lib().aa_paged_evict_workspace_bytes(2, 3, 128, 1000) >= 2 * 3 * 1000 * (4 * 128 + 4)
    assert _hip.lib().aa_paged_evict_workspace_bytes(2, 3, 128, 200) == 0 == _hip.lib().aa_paged_evict_workspace_bytes(64, 8, 128, 10000)  # (rows are moved in turn)
    assert _hip.lib().aa_paged_evict_workspace_bytes(2, 3, 128, 0) == 0 == _hip.lib().aa_paged_evict_workspace_bytes(2, 3, 96, 8)


@pytest.mark.gpu
def test_what_evicting_refuses():
    from anchor_attn.src.ops import _hip
    ops = _ops()
    cache = ops.PagedCache.empty(5, 2, 16, 64, weights=True)
    for t in (cache.keys, cache.values, cache.weights, cache.bounds):
        t.zero_()
    table, lengths = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    good = {"cache": cache, "page_table": table, "lengths": lengths, "n_keys": 8, "n_first": 2, "n_last": 3, "above": 9}
    ops.evict_from_pages(**good)
    twice = torch.zeros(5, 2, 16, 64, dtype=BF16, device="cuda")
    for change in ({"n_keys": 0}, {"n_keys": 4}, {"n_keys": 7.5}, {"n_keys": None}, {"n_keys": (1 << 20) + 1, "above": None}, {"n_first": -1}, {"n_last": -1}, {"n_first": 6}, {"above": 7}, {"above": 1 << 31},
                   {"above": 9.5}, {"page_table": table.long()}, {"page_table": table[:1]}, {"lengths": lengths.cpu()}, {"lengths": [0, 0]}, {"cache": ops.PagedCache(cache.keys, cache.values)},
                   {"cache": ops.PagedCache(twice, twice, None, cache.weights)}, {"cache": 1}):
        with pytest.raises(_hip.AnchorAttnHipError):
            ops.evict_from_pages(**{**good, **change})
    assert ops.evict_from_pages(**{**good, "page_table": table[:0], "lengths": lengths[:0]})[1].shape == (0, 2, 8)
    cache.weights.data = torch.zeros_like(cache.weights)
    with pytest.raises(_hip.AnchorAttnHipError, match="other memory"):
        ops.evict_from_pages(**good)


# ---- together --------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_conversations_that_share_a_prompt_and_give_up_keys():
    """A prompt with norms through the prefill operator and into pages that four conversations share, then steps that append, attend over the shared pages, count
    attention and give up keys behind them; every step against float64 attention over what the cache holds.  The same steps as one captured graph, replayed with eager
    work between, and two such graphs in turn."""
    from anchor_attn.src.ops.anchor_attn_v4 import anchor_attn
    ops = _ops()
    n, batch, hq, hkv, d, page, steps, keep, above = 2048, 4, 8, 2, 128, 64, 6, 2048 + 40, 2048 + 41
    g = torch.Generator(device="cuda").manual_seed(21)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv))
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(BF16) for _ in range(2))
    cos, sin = _tables(4096, d)
    new = [tuple(torch.randn(batch, h, d, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv)) for _ in range(steps)]
    more = {"q_norm": wq, "k_norm": wk}

    def begin():
        s = _Setup([n] + [0] * (batch - 1), hkv, d, page, BF16, 22, room=300)
        own = s.table[:, n // page:n // page + 3].clone()
        s.table[1:, n // page:n // page + 3] = s.table[1:, :3]
        s.table[0, n // page:n // page + 3] = own[0]
        s.table[1:, :n // page] = s.table[0, :n // page]
        s.cache = _weights_of(s)
        k_out = torch.empty_like(k)
        q_out = ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table[:1], _int32([n]), _int32([0, n]), k_out=k_out, **more)
        assert anchor_attn(q_out.transpose(0, 1)[None], k_out.transpose(0, 1)[None], v.transpose(0, 1)[None], return_computational_ratio=False).shape == (1, hq, n, d)
        assert bool((s.cache.weights[s.table[0, :n // page].long()] == 0).all())
        # their own beginnings, of different lengths
        own = [30, 41, 1, 37]
        x = [torch.randn(sum(own), h, d, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(BF16) for h in (hkv, hkv)]
        s.host = [n + m for m in own]
        s.lengths = _int32(s.host)
        ops.append_to_pages(s.cache, None, *x, cos, sin, s.table, s.lengths, _int32([0, 30, 71, 72, 109]), k_norm=wk)
        s.positions, s.roomy = s.lengths.clone(), _roomy(s)
        return s

    shared = _int32([n // page])

    def step(s, x):
        s.lengths += 1
        s.positions += 1
        rotated = ops.append_to_pages(s.cache, *x, cos, sin, s.table, s.lengths, positions=s.positions, **more)
        out = ops.paged_shared_decode_attention(s.cache, rotated, s.roomy, s.lengths, shared)
        same = ops.paged_weighing_decode_attention(s.cache, rotated, s.table, s.lengths, n_first=n)
        had = s.lengths.clone()
        lengths, kept = ops.evict_from_pages(s.cache, s.table, s.lengths, keep, n_first=n, n_last=8, above=above)
        s.lengths.copy_(lengths)
        return rotated, out, same, had, kept, lengths

    s, eager = begin(), []
    prompt = s.cache.keys[s.table[0, :n // page].long()].clone()
    for i, x in enumerate(new):
        outs = step(s, x)
        eager.append([t.clone() for t in outs] + [t.clone() for t in (s.cache.keys, s.cache.values, s.cache.bounds, s.cache.weights)])
    # (each step once more, looked at before keys are given up)
    s = begin()
    gone = 0
    for i, x in enumerate(new):
        s.lengths += 1
        s.positions += 1
        s.host = s.lengths.tolist()
        rotated = ops.append_to_pages(s.cache, *x, cos, sin, s.table, s.lengths, positions=s.positions, **more)
        _near(rotated, x[0], wq, 1e-6, cos[s.positions.long() - 1], sin[s.positions.long() - 1])
        out = ops.paged_shared_decode_attention(s.cache, rotated, s.roomy, s.lengths, shared)
        _close(out, rotated, s, d ** -0.5)
        before = s.cache.weights.clone()
        same = ops.paged_weighing_decode_attention(s.cache, rotated, s.table, s.lengths, n_first=n)
        _close(same, rotated, s, d ** -0.5)
        _weights_close(s.cache.weights, before, rotated, s, d ** -0.5, n)
        assert all(torch.equal(a, b) for a, b in zip((rotated, out, same), eager[i]))
        s.lengths = _evict_and_check(s, s.cache, keep, n, 8, above)
        gone += int(eager[i][3].sum() - s.lengths.sum())
        assert torch.equal(s.lengths, eager[i][5]) and torch.equal(s.cache.keys[s.table[0, :n // page].long()], prompt)
        assert bool((s.cache.weights[s.table[0, :n // page].long()] == 0).all())
    assert gone >= 8 and int((s.positions - s.lengths).sum()) == gone

    graphs = []
    for _ in range(2):
        s, x = begin(), tuple(t.clone() for t in new[0])
        kept_state = [t.clone() for t in (s.lengths, s.positions, s.cache.keys, s.cache.values, s.cache.bounds, s.cache.weights)]
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s, x)  # (warm-up; what it changed is set back)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            outs = step(s, x)
        for a, b in zip((s.lengths, s.positions, s.cache.keys, s.cache.values, s.cache.bounds, s.cache.weights), kept_state):
            a.copy_(b)
        graphs.append((s, x, graph, outs))
    for i in range(steps):
        for s, x, graph, outs in graphs:
            for a, b in zip(x, new[i]):
                a.copy_(b)
            graph.replay()
        step(begin(), new[0])  # (eager work between the replays)
        torch.cuda.synchronize()
        for s, _, _, outs in graphs:
            for a, b in zip((*outs, s.cache.keys, s.cache.values, s.cache.bounds, s.cache.weights), eager[i]):
                assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))


@pytest.mark.gpu
def test_steps_on_two_streams_at_once():
    """Two caches, each on a stream of its own, without waiting in between: the results of one after the other."""
    ops = _ops()

    def begin(seed):
        s, shared, groups = _shared_setup([30, 5], [9, 3], [400, 70, 3], 4, 128, 64, BF16, seed)
        s.cache = _weights_of(s)
        s.cache.weights.zero_()
        s.roomy = _roomy(s)
        return s, s.queries(16), shared, groups

    def work(s, q, shared, groups):
        out = ops.paged_shared_decode_attention(s.cache, q, s.roomy, s.lengths, shared, groups)
        # (one sequence of each group, which share nothing)
        table, lengths = s.table[8:10], s.lengths[8:10]
        weighed = ops.paged_weighing_decode_attention(s.cache, q[8:10], table, lengths)
        return (out, weighed, *ops.evict_from_pages(s.cache, table, lengths, 300, 10, 20), s.cache.keys.clone(), s.cache.weights.clone())

    want = [work(*begin(i)) for i in range(2)]
    mine = [begin(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for x, stream in zip(mine, streams):
        with torch.cuda.stream(stream):
            got.append(work(*x))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0)) for x, y in zip(a, b))
