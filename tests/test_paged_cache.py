"""Appending to a key/value cache in pages and decode steps that read it, whole or sparsely, against plain float64 implementations, at the
lengths, pages and layouts where tiles, pages and shares of the work end.

Tolerances.  u is half a step of the 16-bit type relative to a value (2^-8 for bf16, 2^-11 for fp16).
Rotation: two products and a sum in float32 are off by at most 2^-23 of the products' magnitudes, the rounding by u of the result
(half a step of the subnormals, 2^-25, for fp16).  Bounds are those of the stored keys and have no error.
Attention: a score is a float32 sum of D exact products, off by at most D * 2^-24 * sum |q_d k_d| and twice in a quotient; with its scaling and exp2
(arguments up to 2^8, 2^-24 of them, and an ulp of exp2 or two) a probability is off by 2 * D * 2^-24 * sum |q_d k_d| * scale + 2^-14 of it.  It is kept as two 16-bit numbers,
off by u^2 (fp16: its grid of 2^-39 too, covered by 2^-14); sums over n keys in float32 add n * 2^-24.  All of that is relative to sum p |v| / sum p; the
result is rounded once, u of it.  The chosen pages have to be the same."""
import copy
import ctypes
import pathlib
import pickle
import types

import pytest
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF16, F16 = torch.bfloat16, torch.float16


def _ops():
    from anchor_attn.src.ops import paged_cache
    return paged_cache


def _tables(n, d, base=1e4):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def _pool(n_pages, hkv, page, d, dtype, g, layout):
    """Pool memory in one of three layouts, the rows of its pages contiguous in each."""
    if layout == "heads":  # [pages, KV heads, rows, D]
        return torch.randn(n_pages, hkv, page, d, generator=g, device="cuda").to(dtype)
    if layout == "rows":  # [pages, rows, KV heads, D]
        return torch.randn(n_pages, page, hkv, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
    wide = torch.randn(n_pages, hkv + 1, page + 3, d + 8, generator=g, device="cuda").to(dtype)  # a part of something larger
    return wide[:, 1:, 2:2 + page, 8:]


class _Setup:
    """A cache with keys of ``lengths`` in pages in random order; NaN where no sequence has a key; bounds of what is there."""

    def __init__(self, lengths, hkv, d, page, dtype, seed, layout="heads", room=0, extra=0):
        self.g = g = torch.Generator(device="cuda").manual_seed(seed)
        self.page, self.d, self.hkv, self.dtype, self.host = page, d, hkv, dtype, list(lengths)
        counts = [(n + room + page - 1) // page for n in lengths]
        total = sum(counts) + 3
        keys, values = (_pool(total, hkv, page, d, dtype, g, layout) for _ in range(2))
        order = torch.randperm(total, generator=g, device="cuda").int()
        self.table = torch.full((len(lengths), max(1, max(counts, default=1)) + extra), -1, dtype=torch.int32, device="cuda")
        self.table[:, 1::2] = 2 ** 31 - 1  # (what is behind a sequence's pages does not matter)
        used = torch.zeros(total, dtype=torch.int64, device="cuda")
        begin = 0
        for b, (n, c) in enumerate(zip(lengths, counts)):
            mine = order[begin:begin + c]
            self.table[b, :c] = mine
            used[mine.long()] = (n - page * torch.arange(c, device="cuda")).clamp(0, page)
            begin += c
        there = (torch.arange(page, device="cuda") < used[:, None])[:, None, :, None]
        keys.masked_fill_(~there, float("nan"))
        values.masked_fill_(~there, float("nan"))
        lo = torch.where(there, keys, float("inf")).amin(2)
        hi = torch.where(there, keys, float("-inf")).amax(2)
        bounds = torch.stack((lo, hi), 2).masked_fill((used == 0)[:, None, None, None], float("nan")).contiguous()
        self.cache = _ops().PagedCache(keys, values, bounds)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def rows(self, pool, b, h, pages=None):
        """Keys or values of a sequence and KV head in order, float64 (of some pages, counted in the sequence)."""
        n = self.host[b]
        there = (n + self.page - 1) // self.page
        pages = torch.arange(there, device="cuda") if pages is None else pages
        last = there - 1
        x = pool[self.table[b, pages].long(), h].reshape(-1, self.d)
        return x[:x.shape[0] - (there * self.page - n)].double() if last >= 0 else x[:0].double()

    def queries(self, hq, spread=3.0):
        return (spread * torch.randn(len(self.host), hq, self.d, generator=self.g, device="cuda")).to(self.dtype)


def _close(out, q, s, scale, pages=None):
    dtype, d = out.dtype, s.d
    group = q.shape[1] // s.hkv
    for b in range(q.shape[0]):
        for h in range(s.hkv):
            got = out[b, h * group:(h + 1) * group].double()
            if s.host[b] == 0:
                assert bool((got == 0).all())
                continue
            mine = None if pages is None else pages[b, h][pages[b, h] >= 0].long()
            k, v = s.rows(s.cache.keys, b, h, mine), s.rows(s.cache.values, b, h, mine)
            x = q[b, h * group:(h + 1) * group].double()
            p = (x @ k.T * scale).softmax(-1)
            want = p @ v
            magnitude = (x.abs() @ k.abs().T).amax(-1, keepdim=True) * scale
            relative = 2.0 * d * 2.0 ** -24 * magnitude + 2.0 ** -14 + U[dtype] ** 2 + k.shape[0] * 2.0 ** -24
            bound = U[dtype] * want.abs() * 1.001 + relative * (p @ v.abs()) + 2.0 ** -25
            err = (got - want).abs()
            assert bool((err <= bound).all()), (b, h, float((err - bound).max()), float(err.max()))


def _chosen(q, s, n_pages, n_first, n_last):
    """The pages by their definition: scores in float64, rounded to float32, sorted on the host."""
    group = q.shape[1] // s.hkv
    got = torch.full((q.shape[0], s.hkv, n_pages), -1, dtype=torch.int32)
    for b in range(q.shape[0]):
        there = (s.host[b] + s.page - 1) // s.page
        at = s.table[b, :there].long()
        for h in range(s.hkv):
            if there <= n_pages:
                got[b, h, :there] = torch.arange(there, dtype=torch.int32)
                continue
            lo, hi = s.cache.bounds[at, h].double().unbind(1)
            x = q[b, h * group:(h + 1) * group, None].double()
            score = torch.where(x >= 0, x * hi, x * lo).sum(-1).amax(0).float().tolist()
            score = [float("inf") if x != x else x for x in score]
            ends = set(range(n_first)) | set(range(there - n_last, there))
            rank = sorted((i for i in range(there) if i not in ends), key=lambda i: (-score[i], i))
            got[b, h] = torch.tensor(sorted(ends | set(rank[:n_pages - len(ends)])), dtype=torch.int32)
    return got.cuda()


def _rotated(x, cos, sin):
    """Float64 rotation of ``[tokens, heads, D]`` by rows of the tables, and the magnitude that errors are relative to."""
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half].double(), x[..., half:].double(), cos.double()[:, None], sin.double()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), -1), torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)


def _rounded(got, want, magnitude):
    err = (got.double() - want).abs()
    bound = U[got.dtype] * want.abs() * 1.001 + 2.0 ** -23 * magnitude + 2.0 ** -25
    assert bool((err <= bound).all()), float((err - bound).max())


# ---- appending -----------------------------------------------------------------------------------------------------

def _append_and_check(before, new, hq, hkv, d, page, dtype, layout, steps=False, padding=0, seed=0, bounds=True):
    ops = _ops()
    s = _Setup(before, hkv, d, page, dtype, seed, layout, room=max(new))
    n = sum(new)
    parts = (torch.randn(n + padding, hq + 2 * hkv, d, generator=s.g, device="cuda") * 2).to(dtype)
    q, k, v = parts.split((hq, hkv, hkv), 1)
    lengths = [a + b for a, b in zip(before, new)]
    cos, sin = _tables(max(lengths) + 1, d)
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    cache = s.cache if bounds else ops.PagedCache(s.cache.keys, s.cache.values)
    keys, values, old = s.cache.keys.clone(), s.cache.values.clone(), s.cache.bounds.clone()
    out = torch.full((n + padding, hq, d), 7.0, dtype=dtype, device="cuda")
    got = ops.append_to_pages(cache, q, k, v, cos, sin, s.table, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                              None if steps else torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    assert got is out and bool((out[n:] == 7.0).all())
    positions = torch.tensor([p for a, b in zip(before, new) for p in range(a, a + b)], device="cuda")
    sequence = torch.tensor([i for i, b in enumerate(new) for _ in range(b)], device="cuda")
    if n:
        _rounded(out[:n], *_rotated(q[:n], cos[positions], sin[positions]))
        at, slot = s.table[sequence, positions // page].long(), positions % page
        stored = s.cache.keys[at, :, slot]
        _rounded(stored, *_rotated(k[:n], cos[positions], sin[positions]))
        assert torch.equal(s.cache.values[at, :, slot], v[:n])
        keys[at, :, slot], values[at, :, slot] = stored, v[:n]
    # nothing else has changed
    for x, y in ((s.cache.keys, keys), (s.cache.values, values)):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))
    if bounds:
        for b, (a, c) in enumerate(zip(before, new)):
            for i in range(a // page, (a + c + page - 1) // page if c else 0):
                page_keys = s.cache.keys[int(s.table[b, i]), :, :min(page, a + c - i * page)]
                old[int(s.table[b, i])] = torch.stack((page_keys.amin(1), page_keys.amax(1)), 1)
    assert torch.equal(s.cache.bounds.nan_to_num(9.0), old.nan_to_num(9.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("before,new,hq,hkv,d,page,layout,padding", [
    ([0], [1], 32, 8, 128, 64, "heads", 0),
    ([0, 63, 64, 17], [130, 1, 64, 0], 28, 4, 128, 64, "rows", 5),
    ([5, 0, 31, 100], [1, 33, 2, 300], 14, 2, 64, 16, "heads", 0),
    ([0, 1, 255, 256], [257, 600, 1, 255], 8, 8, 128, 256, "part", 0),
    ([0] * 70, [3] * 69 + [40], 4, 1, 64, 32, "heads", 70),
    ([7, 128], [0, 0], 4, 2, 128, 128, "heads", 3),
    ([7] * 4, [9, 0, 1, 70], 4, 2, 128, 32, "heads", 3),
    ([2, 5] + [0] * 200 + [9, 1], [1, 2] + [0] * 200 + [30, 1], 4, 1, 128, 16, "heads", 40),
    ([3] * 300 + [0] * 4400, [i % 3 for i in range(300)] + [0] * 4000 + [1, 0, 0, 2] * 100, 2, 1, 64, 16, "heads", 11),
    ([300] * 3, [517, 1, 90], 71, 1, 64, 128, "part", 1),
])
def test_append(before, new, hq, hkv, d, page, layout, padding, dtype):
    _append_and_check(before, new, hq, hkv, d, page, dtype, layout, padding=padding, seed=len(before))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,hq,hkv,d,page,bounds", [(1, 32, 8, 128, 64, True), (97, 28, 4, 128, 16, True), (33, 32, 8, 64, 256, False), (300, 14, 2, 64, 32, True)])
def test_append_one_token_each(batch, hq, hkv, d, page, bounds):
    _append_and_check([(37 * b) % 211 for b in range(batch)], [1] * batch, hq, hkv, d, page, BF16, "heads", steps=True, seed=batch, bounds=bounds)


@pytest.mark.gpu
def test_append_without_rotation_and_in_place():
    ops = _ops()
    s = _Setup([3, 40], 2, 64, 16, BF16, 4, room=9)
    k, v, q = (torch.randn(18, h, 64, generator=s.g, device="cuda").to(BF16) for h in (2, 2, 6))
    starts, lengths = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 9, 18], [12, 49]))
    assert ops.append_to_pages(s.cache, None, k, v, None, None, s.table, lengths, starts) is None
    s.host = [12, 49]
    for b in range(2):
        for h in range(2):
            assert torch.equal(s.rows(s.cache.keys, b, h)[-9:], k[9 * b:9 * b + 9, h].double())
            assert torch.equal(s.rows(s.cache.values, b, h)[-9:], v[9 * b:9 * b + 9, h].double())
    cos, sin = torch.cat(_tables(64, 64), 1).split(32, 1)  # (parts of one table)
    want = ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table, lengths, starts)
    assert torch.equal(want, ops.append_to_pages(s.cache, q, k, v, cos.contiguous(), sin.contiguous(), s.table, lengths, starts))
    keys = s.cache.keys.clone()
    assert ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table, lengths, starts, out=q) is q
    assert torch.equal(q, want) and torch.equal(keys.nan_to_num(9.0), s.cache.keys.nan_to_num(9.0))


@pytest.mark.gpu
def test_tokens_without_a_place_are_left_out():
    """A length of 0, positions below 0 and behind the angles, the table or the pool's pages, starts beyond the tokens."""
    ops = _ops()
    s = _Setup([0] * 6, 2, 64, 16, BF16, 5, room=40)
    keys, values, bounds = s.cache.keys.clone(), s.cache.values.clone(), s.cache.bounds.clone()
    q, k, v = (torch.randn(6, h, 64, generator=s.g, device="cuda").to(BF16) for h in (4, 2, 2))
    cos, sin = _tables(40, 64)
    s.table[3, 0], s.table[4, 0] = -1, s.cache.n_pages
    lengths = torch.tensor([0, 41, 1000, 5, 5, -7], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table, lengths, out=out)
    assert bool((out == 7.0).all())
    # one sequence of six tokens whose length is 2: the first four have positions below 0; and one whose tokens end behind the last
    for begins, n, placed in (([0, 6, 6, 6, 6, 6, 6], 2, [4, 5]), ([6, 6, 6, 6, 6, 6, 6], 2, []), ([0, 3, 2 ** 31 - 1, 6, 6, 6, 6], 3, [0, 1, 2])):
        for x, y in ((s.cache.keys, keys), (s.cache.values, values), (s.cache.bounds, bounds)):
            x.copy_(y)
        lengths = torch.tensor([n] + [0] * 5, dtype=torch.int32, device="cuda")
        out = ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table, lengths, torch.tensor(begins, dtype=torch.int32, device="cuda"), out=torch.full_like(q, 7.0))
        assert [i for i in range(6) if bool((out[i] != 7.0).any())] == placed
        assert int((~s.cache.keys.isnan()).sum()) == len(placed) * 2 * 64 == int((~s.cache.values.isnan()).sum())


@pytest.mark.gpu
def test_bounds_of_infinite_and_nan_keys():
    ops = _ops()
    s = _Setup([0], 1, 64, 16, F16, 6, room=32)
    k = torch.randn(20, 1, 64, generator=s.g, device="cuda").to(F16)
    k[3, 0, 5], k[4, 0, 6], k[5, 0, 7], k[17, 0, 8], k[18, 0, 9], k[19, 0, 10], k[6, 0, 11] = float("nan"), float("inf"), float("-inf"), float("nan"), 65504.0, -float("nan"), -0.0
    for lo, hi, length in ((0, 17, 17), (17, 20, 20)):
        ops.append_to_pages(s.cache, None, k[lo:hi], k[lo:hi], None, None, s.table, torch.tensor([length], dtype=torch.int32, device="cuda"),
                            torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"))
    for i, rows in enumerate((k[:16, 0], k[16:, 0])):
        got = s.cache.bounds[int(s.table[0, i]), 0]
        want = torch.stack((rows.amin(0), rows.amax(0)))  # (the framework's minimum of NaN is NaN)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0))


# ---- reading -------------------------------------------------------------------------------------------------------

LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 500, 1023]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hq,hkv,d,page,layout", [
    (LENGTHS, 32, 8, 128, 64, "heads"), (LENGTHS, 28, 4, 128, 16, "rows"), (LENGTHS, 14, 2, 64, 16, "heads"), (LENGTHS, 32, 8, 64, 32, "part"),
    (LENGTHS, 3, 3, 128, 256, "heads"), ([700, 1, 33], 16, 1, 64, 128, "heads"), ([700, 1, 33], 17, 1, 128, 128, "rows"), ([900, 0], 71, 1, 64, 64, "heads"),
    ([20001], 32, 8, 128, 64, "heads"), ([9000, 40, 12345], 28, 4, 64, 16, "heads"), ([5], 14, 2, 64, 16, "heads"), ([0], 4, 2, 128, 16, "heads"),
    ([70001], 8, 1, 128, 256, "rows"), ([700] * 130 + [5000], 8, 2, 64, 64, "heads"), ([2500, 0, 0, 1] * 30, 4, 1, 64, 32, "heads"), ([700, 650, 641, 640, 639] * 60, 2, 2, 64, 32, "heads"), ([1] * 300, 14, 2, 64, 16, "heads"), ([33, 7] * 500, 4, 1, 128, 32, "heads"), ([4097] + [3] * 63, 8, 2, 128, 64, "heads"),
])
def test_decode(lengths, hq, hkv, d, page, layout, dtype):
    s = _Setup(lengths, hkv, d, page, dtype, hq + page, layout, extra=hq % 3)
    q = s.queries(hq)
    wide = torch.full((len(lengths), hq + 1, d + 8), 7.0, dtype=dtype, device="cuda")
    out = wide[:, 1:, 8:]
    assert _ops().paged_decode_attention(s.cache, q, s.table, s.lengths, out=out) is out
    assert bool((wide[:, 0] == 7.0).all()) and bool((wide[:, :, :8] == 7.0).all())
    _close(out, q, s, d ** -0.5)
    again = _ops().paged_decode_attention(s.cache, q.transpose(0, 1).contiguous().transpose(0, 1), s.table, s.lengths, sm_scale=d ** -0.5)
    assert torch.equal(out, again)  # the same bits
    assert _ops().paged_decode_attention(s.cache, q, s.table, s.lengths, out=q) is q and torch.equal(q, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_with_an_attention_sink_and_a_scale(dtype):
    """One key far above the others, whose probabilities lie on the 16-bit types' lowest grid."""
    s = _Setup([6000, 300], 2, 128, 64, dtype, 3)
    q = s.queries(8, 1.0)
    q[:, :, 0] = 8.0
    for b in range(2):
        s.cache.keys[s.table[b, 0].long(), :, 0, 0] = 16.0
    for scale in (0.088, 0.01, 1.0):
        _close(_ops().paged_decode_attention(s.cache, q, s.table, s.lengths, sm_scale=scale), q, s, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("length,d", [(40, 128), (5000, 64)])
def test_decode_with_infinite_and_nan_values_that_are_seen(length, d, dtype):
    """An infinite value gives an infinity in its channel, NaN gives NaN, and the other channels stay as they are."""
    s = _Setup([length], 2, d, 16, dtype, 8)
    q = s.queries(8, 0.3)
    want = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    at = s.table[0, 1].long()
    s.cache.values[at, 0, 3, 5], s.cache.values[at, 0, 4, 6], s.cache.values[at, 0, 9, 7] = float("inf"), float("-inf"), float("nan")
    s.cache.values[at, 0, 3, 8], s.cache.values[at, 0, 4, 8] = float("inf"), float("-inf")
    got = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    assert bool((got[0, :4, 5] == float("inf")).all()) and bool((got[0, :4, 6] == float("-inf")).all()) and bool(got[0, :4, 7:9].isnan().all())
    assert torch.equal(got[0, 4:], want[0, 4:])
    rest = torch.ones(d, dtype=torch.bool, device="cuda")
    rest[5:9] = False
    assert bool(((got[0, :4, rest] - want[0, :4, rest]).abs() <= 2 * U[dtype] * want[0, :4, rest].abs() + 2.0 ** -13).all())


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_decode_with_nan_and_infinite_keys(what):
    """A NaN score, or one of plus infinity, makes its heads NaN, as a soft-max in float32 has it, and no others; minus infinity leaves the key out."""
    s = _Setup([100, 100], 2, 64, 16, BF16, 9)
    q = s.queries(4, 0.5)
    q[:, :, 0] = 1.0
    want = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    s.cache.keys[s.table[0, 2].long(), 0, 1, 0] = float(what)
    got = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    assert bool(got[0, :2].isnan().all()) and torch.equal(got[0, 2:], want[0, 2:]) and torch.equal(got[1], want[1])
    s.cache.keys[s.table[0, 2].long(), 0, 1, 0] = float("-inf")
    got = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    assert bool(got.isfinite().all()) and torch.equal(got[0, 2:], want[0, 2:])


@pytest.mark.gpu
def test_lengths_and_pages_that_do_not_fit_are_clamped():
    """Lengths above the table are its size, pages outside the pool the nearest one; nothing else is read."""
    s = _Setup([64, 64, 64], 2, 64, 16, BF16, 10)
    q = s.queries(4)
    want = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    lengths = torch.tensor([1000, 64, -3], dtype=torch.int32, device="cuda")
    got = _ops().paged_decode_attention(s.cache, q, s.table, lengths)
    assert torch.equal(got[:2], want[:2]) and bool((got[2] == 0).all())
    table = s.table.clone()
    s.cache.keys.nan_to_num_(0.5), s.cache.values.nan_to_num_(0.5), s.cache.bounds.nan_to_num_(0.5)
    table[1, 2], table[1, 3] = -5, 2 ** 31 - 1
    s.table[1, 2], s.table[1, 3] = 0, s.cache.n_pages - 1
    assert torch.equal(_ops().paged_decode_attention(s.cache, q, table, lengths), _ops().paged_decode_attention(s.cache, q, s.table, lengths))
    for a, b in zip(*(_ops().paged_sparse_decode_attention(s.cache, q, t, lengths, 3) for t in (table, s.table))):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_pools_beyond_four_gib(dtype):
    ops = _ops()
    n_pages = (9 << 30) // (8 * 64 * 128 * 2)
    s = _Setup([200, 129], 8, 128, 64, dtype, 11)
    small, table = s.cache, s.table.clone()
    big = ops.PagedCache.empty(n_pages, 8, 64, 128, dtype)
    place = n_pages - 1 - 7 * torch.arange(small.n_pages, device="cuda")
    for a, b in ((big.keys, small.keys), (big.values, small.values), (big.bounds, small.bounds)):
        a[place] = b
    q = s.queries(32)
    big_table = torch.where((table >= 0) & (table < small.n_pages), place[table.clamp(0, small.n_pages - 1).long()].int(), -1)
    assert torch.equal(ops.paged_decode_attention(small, q, table, s.lengths), ops.paged_decode_attention(big, q, big_table, s.lengths))
    for a, b in zip(ops.paged_sparse_decode_attention(small, q, table, s.lengths, 2), ops.paged_sparse_decode_attention(big, q, big_table, s.lengths, 2)):
        assert torch.equal(a, b)
    cos, sin = _tables(256, 128)
    k, v = (torch.randn(2, 8, 128, device="cuda").to(dtype) for _ in range(2))
    s.lengths.sub_(1)
    for cache, t in ((small, table), (big, big_table)):
        ops.append_to_pages(cache, q, k, v, cos, sin, t, s.lengths)
    for a, b in ((big.keys, small.keys), (big.values, small.values), (big.bounds, small.bounds)):
        assert torch.equal(a[place].nan_to_num(9.0), b.nan_to_num(9.0))


# ---- sparse reading ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hq,hkv,d,page,n_pages,n_first,n_last", [
    (LENGTHS, 32, 8, 128, 16, 5, 1, 1), (LENGTHS, 28, 4, 64, 16, 8, 0, 3), ([1000, 999, 17], 14, 2, 64, 32, 6, 2, 4), ([1000, 0], 3, 3, 128, 256, 1, 0, 1),
    ([20001], 32, 8, 128, 64, 33, 1, 2), ([60000, 3000], 8, 1, 64, 16, 200, 1, 2), ([2100], 14, 2, 64, 16, 32, 1, 2), ([800] * 40, 4, 2, 64, 16, 9, 1, 1),
    ([5000, 70], 71, 1, 128, 32, 20, 1, 1), ([300, 40], 16, 1, 64, 64, 100, 1, 1), ([1 << 17], 4, 1, 64, 16, 500, 3, 3),
    ([1 << 19, 9], 2, 1, 64, 16, 300, 1, 1), ([16 * 2048], 4, 2, 64, 16, 70, 1, 2), ([16 * 2049 - 5, 3000], 4, 2, 64, 16, 1500, 0, 2), ([16 * 4099, 16 * 4096], 2, 2, 64, 16, 2000, 7, 5),
])
def test_sparse_decode(lengths, hq, hkv, d, page, n_pages, n_first, n_last, dtype):
    s = _Setup(lengths, hkv, d, page, dtype, hq + n_pages, extra=1)
    q = s.queries(hq)
    out, pages = _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n_pages, n_first, n_last)
    assert torch.equal(pages, _chosen(q, s, n_pages, n_first, n_last))
    _close(out, q, s, d ** -0.5, pages)


@pytest.mark.gpu
def test_equal_scores_go_to_the_lower_page():
    for d, dtype, hkv, group in ((64, BF16, 2, 2), (128, F16, 1, 7)):
        s = _Setup([16 * 100, 16 * 700], hkv, d, 16, dtype, 12)
        s.cache.keys.copy_(torch.randn(d, generator=s.g, device="cuda").to(dtype).expand_as(s.cache.keys))
        s.cache.bounds.copy_(s.cache.keys[:, :, :2])
        # a few pages stand out, two of them alike
        for i, f in ((50, 3.0), (20, 2.0), (70, 2.0), (30, 1.5)):
            s.cache.bounds[s.table[:, i].long(), :, 1] = f * s.cache.bounds[0, 0, 1].abs().max() + 1
        q = s.queries(hkv * group).abs()
        for n in (3, 4, 5, 6, 7, 40):
            got = _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n, 1, 1)[1]
            assert torch.equal(got, _chosen(q, s, n, 1, 1))


@pytest.mark.gpu
def test_scores_that_are_nan_or_infinite_come_first():
    s = _Setup([16 * 60], 1, 64, 16, BF16, 13)
    q = s.queries(2)
    q[0, :, 1:4] = 1.0
    at = s.table[0].long()
    s.cache.bounds[at[40], 0, 1, 1], s.cache.bounds[at[30], 0, 0, 2], s.cache.bounds[at[20], 0, :, 3] = float("inf"), float("nan"), float("nan")
    s.cache.bounds[at[10], 0, 1, 3] = float("-inf")
    q[0, 1, 4] = -0.0
    s.cache.bounds[at[:], 0, 0, 4] = float("-inf")  # (-0 is not below 0: the larger bound counts)
    q[0, 0, 4] = 0.0
    for n in (3, 4, 5, 30, 58, 59):
        assert torch.equal(_ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n, 1, 1)[1], _chosen(q, s, n, 1, 1))


# ---- together ------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_a_prompt_and_decode_steps_together():
    """A prompt through the prefill operator and into pages, then steps that append and attend; the same steps once more as one captured graph, with a
    second graph in between that another cache's step was captured into.  Every step against float64 attention over what the cache holds."""
    from anchor_attn.src.ops.anchor_attn_v4 import anchor_attn
    ops = _ops()
    n, hq, hkv, d, page, steps = 2048, 8, 2, 128, 64, 4
    g = torch.Generator(device="cuda").manual_seed(21)
    q, k, v = (torch.randn(1, n, h, d, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv))
    assert anchor_attn(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), return_computational_ratio=False).shape == (1, hq, n, d)
    cos, sin = _tables(4096, d)

    def begin():
        s = _Setup([0, 0], hkv, d, page, BF16, 22, room=n + 200)
        s.table[1, :20] = s.table[1, :20].flip(0)
        prompt = torch.tensor([n, 129], dtype=torch.int32, device="cuda")
        ops.append_to_pages(s.cache, None, torch.cat((k[0], k[0, :129])), torch.cat((v[0], v[0, :129])), None, None, s.table, prompt,
                            torch.tensor([0, n, n + 129], dtype=torch.int32, device="cuda"))
        s.lengths = prompt
        return s

    new = [tuple(torch.randn(2, h, d, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv)) for _ in range(steps)]

    def step(s, x):
        s.lengths += 1
        rotated = ops.append_to_pages(s.cache, *x, cos, sin, s.table, s.lengths)
        return (rotated, ops.paged_decode_attention(s.cache, rotated, s.table, s.lengths), *ops.paged_sparse_decode_attention(s.cache, rotated, s.table, s.lengths, 8, 1, 2))

    s, eager = begin(), []
    for i, x in enumerate(new):
        rotated, out, sparse, pages = step(s, x)
        s.host = [n + i + 1, 129 + i + 1]
        _close(out, rotated, s, d ** -0.5)
        assert torch.equal(pages, _chosen(rotated, s, 8, 1, 2))
        _close(sparse, rotated, s, d ** -0.5, pages)
        eager.append([t.clone() for t in (rotated, out, sparse, pages)])

    graphs = []
    for _ in range(2):
        s, x = begin(), tuple(t.clone() for t in new[0])
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s, x)  # (warm-up; the lengths are set back)
        torch.cuda.current_stream().wait_stream(side)
        s.lengths -= 1
        with torch.cuda.graph(graph):
            outs = step(s, x)
        graphs.append((s, x, graph, outs))
    for i in range(steps):
        for s, x, graph, outs in graphs:
            for a, b in zip(x, new[i]):
                a.copy_(b)
            graph.replay()
        step(begin(), new[0])  # (eager work between the replays)
        torch.cuda.synchronize()
        for _, _, _, outs in graphs:
            for a, b in zip(outs, eager[i]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once():
    ops = _ops()
    s = _Setup([3000, 5000, 100], 4, 128, 64, BF16, 31)
    q = [s.queries(16) for _ in range(2)]
    want = [(ops.paged_decode_attention(s.cache, x, s.table, s.lengths), *ops.paged_sparse_decode_attention(s.cache, x, s.table, s.lengths, 9)) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append((ops.paged_decode_attention(s.cache, q[i], s.table, s.lengths), *ops.paged_sparse_decode_attention(s.cache, q[i], s.table, s.lengths, 9)))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


# ---- refusals ------------------------------------------------------------------------------------------------------

CACHE = {"keys": 4096, "kp_sp": 4096, "kp_sh": 2048, "kp_sn": 128, "values": 4096, "vp_sp": 4096, "vp_sh": 2048, "vp_sn": 128, "bounds": 4096,
         "n_pages": 9, "n_kv_heads": 2, "page_size": 16, "head_dim": 128, "dtype": 0}
TOKENS = {"q": 4096, "q_st": 1024, "q_sh": 128, "q_out": 4096, "qo_st": 1024, "qo_sh": 128, "k": 4096, "k_st": 256, "k_sh": 128, "v": 4096, "v_st": 256, "v_sh": 128,
          "cos": 4096, "sin": 4096, "cs_sn": 64, "page_table": 4096, "pt_sb": 8, "lengths": 4096, "starts": 4096, "n_positions": 100, "batch": 2, "n_tokens": 5, "n_q_heads": 8,
          "max_pages": 8}
STEP = {"q": 4096, "q_sb": 1024, "q_sh": 128, "out": 4096, "o_sb": 1024, "o_sh": 128, "page_table": 4096, "pt_sb": 8, "lengths": 4096, "workspace": 4096,
        "workspace_bytes": 1 << 40, "pages": 4096, "batch": 2, "n_q_heads": 8, "max_pages": 100, "n_chosen": 4, "n_first": 1, "n_last": 1, "sm_scale": 0.1}
EVERY = [({"batch": 0}, "must be positive"), ({"batch": 65536}, "not supported"), ({"n_kv_heads": 3}, "must divide"), ({"n_kv_heads": 0}, "must be positive"),
         ({"head_dim": 96}, "head_dim 96"), ({"page_size": 48}, "page_size 48"), ({"page_size": 8}, "page_size 8"), ({"n_pages": 0}, "must be positive"),
         ({"max_pages": 0}, "must be positive"), ({"max_pages": 65537}, "not supported"), ({"dtype": 2}, "dtype"), ({"keys": 0}, "keys is NULL"),
         ({"keys": 4104}, "keys must be 16-byte aligned"), ({"kp_sh": 2052}, "keys must be 16-byte aligned"), ({"vp_sn": 120}, "smaller than head_dim"),
         ({"vp_sn": 16392}, "larger than 16384"), ({"values": 0}, "values is NULL"), ({"page_table": 0}, "page_table is NULL"), ({"lengths": 0}, "lengths is NULL"),
         ({"lengths": 4098}, "lengths must be 4-byte aligned"), ({"q": 4104}, "q must be 16-byte aligned"), ({"q_sh": 60}, "q must have strides"),
         ({"bounds": 8}, "bounds must be 16-byte"), ({"cache": None}, "cache is NULL"), ({"given": None}, "is NULL")]
READ = [({"q": 0}, "q is NULL"), ({"out": 0}, "out is NULL"), ({"out": 8}, "out must be 16-byte"), ({"sm_scale": 0.0}, "sm_scale"), ({"sm_scale": float("nan")}, "sm_scale"),
        ({"sm_scale": float("inf")}, "sm_scale"), ({"n_q_heads": 0}, "query heads"), ({"batch": 4096, "n_q_heads": 4096}, "together")]


@pytest.mark.parametrize("fn,change,message", [
    *[("append", c, m) for c, m in EVERY], *[("decode", c, m) for c, m in EVERY + READ], *[("sparse", c, m) for c, m in EVERY + READ],
    ("append", {"n_tokens": 0}, "0 tokens"), ("append", {"n_tokens": 1 << 24}, "not supported"), ("append", {"n_tokens": 1 << 22}, "not supported"), ("decode", {"workspace_bytes": 100}, "workspace has 100 bytes"), ("decode", {"workspace": 0}, "workspace is NULL"), ("append", {"starts": 0}, "5 tokens of 2 sequences"),
    ("append", {"cos": 0}, "come together"), ("append", {"q": 0}, "come together"), ("append", {"q_out": 0}, "come together"), ("append", {"cos": 0, "sin": 0}, "come together"),
    ("append", {"n_q_heads": 0}, "come together"), ("append", {"cs_sn": 63}, "cos and sin"), ("append", {"cs_sn": 60}, "cos and sin"), ("append", {"n_positions": 0}, "cos and sin"),
    ("append", {"sin": 4100}, "sin must be 16-byte"), ("append", {"k": 0}, "k is NULL"), ("append", {"v": 4}, "v must be 16-byte"), ("append", {"v_st": 4}, "v must have strides"),
    ("append", {"starts": 6}, "starts must be 4-byte"),
    ("sparse", {"n_last": 0}, "at least the last one"), ("sparse", {"n_first": -1}, "not supported"), ("sparse", {"n_first": 4}, "not supported"),
    ("sparse", {"n_chosen": 65537}, "not supported"), ("sparse", {"n_chosen": 1}, "not supported"), ("sparse", {"bounds": 0}, "bounds is NULL"),
    ("sparse", {"pages": 0}, "pages is NULL"), ("sparse", {"workspace_bytes": 100}, "workspace has 100 bytes"), ("sparse", {"workspace": 0}, "workspace is NULL"),
])
def test_what_the_c_interface_refuses(fn, change, message):
    """Before anything is launched: the addresses are never read."""
    from anchor_attn.src.ops import _hip
    lib = _hip.lib()
    given, packs, f = {"append": (TOKENS, _hip.PAGED_TOKENS, lib.aa_paged_append), "decode": (STEP, _hip.PAGED_STEP, lib.aa_paged_decode_fwd),
                       "sparse": (STEP, _hip.PAGED_STEP, lib.aa_paged_sparse_decode_fwd)}[fn]
    assert set(change) <= {*given, *CACHE, "cache", "given"}
    struct = _hip.PagedCacheStruct(*{**CACHE, **{k: v for k, v in change.items() if k in CACHE}}.values())
    with pytest.raises(_hip.AnchorAttnHipError, match=message):
        _hip.check(f(None if "cache" in change else ctypes.addressof(struct),
                     None if "given" in change else packs.pack(*{**given, **{k: v for k, v in change.items() if k in given}}.values()), None))


def test_packed_structs_are_laid_out_as_in_c(tmp_path):
    import subprocess
    from anchor_attn.src.ops import _hip
    source = tmp_path / "sizes.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "anchor_attn_hip.h"\nint main(void) { printf("%zu %zu %zu %zu %zu", sizeof(aa_paged_cache), '
                      'sizeof(aa_paged_tokens), sizeof(aa_paged_step), offsetof(aa_paged_tokens, n_positions), offsetof(aa_paged_step, sm_scale)); return 0; }\n')
    include = pathlib.Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", f"-I{include}", "-o", tmp_path / "sizes", source], check=True)
    sizes = [int(x) for x in subprocess.run([tmp_path / "sizes"], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes[:3] == [ctypes.sizeof(_hip.PagedCacheStruct), _hip.PAGED_TOKENS.size, _hip.PAGED_STEP.size]
    assert _hip.PAGED_TOKENS.pack(*range(24))[sizes[3]] == 19 and _hip.PAGED_STEP.pack(*[0] * 18, 1.0)[sizes[4]:][:4] == b"\0\0\x80?"


def test_caches_that_are_refused():
    from anchor_attn.src.ops import _hip
    x = torch.zeros(3, 2, 16, 64, dtype=BF16)
    with pytest.raises(_hip.AnchorAttnHipError, match="one GPU"):
        _ops().PagedCache(x, x)
    with pytest.raises(_hip.AnchorAttnHipError, match="must be a PagedCache"):
        _ops().paged_decode_attention(types.SimpleNamespace(), x, x, x)


@pytest.mark.gpu
def test_what_the_entry_points_refuse():
    from anchor_attn.src.ops import _hip
    ops = _ops()
    z = lambda *shape, dtype=BF16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    for keys, values, bounds in ((z(3, 2, 16, 64), z(3, 2, 16, 128), None), (z(3, 2, 24, 64), z(3, 2, 24, 64), None), (z(3, 2, 16, 96), z(3, 2, 16, 96), None),
                                 (z(3, 2, 16, 64, dtype=torch.float32),) * 2 + (None,), (z(3, 2, 16, 64), z(3, 2, 16, 64, dtype=F16), None),
                                 (z(3, 2, 16, 64), z(3, 2, 16, 64), z(3, 2, 2, 128)), (z(3, 2, 16, 64), z(3, 2, 16, 64), z(2, 3, 2, 64).transpose(0, 1)),
                                 (z(3, 2, 16, 128)[..., ::2], z(3, 2, 16, 64), None), (z(3, 2, 16, 68)[..., 4:], z(3, 2, 16, 64), None), (z(0, 2, 16, 64),) * 2 + (None,),
                                 (z(3, 2, 16, 64).requires_grad_(), z(3, 2, 16, 64), None), (z(1, 2, 1, 64).expand(3, 2, 16, 64), z(3, 2, 16, 64), None)):
        with pytest.raises(_hip.AnchorAttnHipError):
            ops.PagedCache(keys, values, bounds)
    cache = ops.PagedCache.empty(5, 2, 16, 64)
    table, lengths, starts = z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), z(3, dtype=torch.int32)
    q, k, v, cos = z(2, 4, 64), z(2, 2, 64), z(2, 2, 64), z(50, 32, dtype=torch.float32)
    good = {"cache": cache, "q": q, "page_table": table, "lengths": lengths}
    more = {**good, "k": k, "v": v, "cos": cos, "sin": cos, "starts": starts}
    reads = [{"q": z(2, 3, 64)}, {"q": z(3, 4, 64)}, {"q": z(2, 4, 128)}, {"q": z(2, 4, 64, dtype=F16)}, {"q": z(2, 64)}, {"q": z(2, 4, 128)[..., ::2]}, {"q": q.cpu()},
             {"q": z(2, 4, 64).requires_grad_()}, {"page_table": table.long()}, {"page_table": table[0]}, {"page_table": z(3, 3, dtype=torch.int32)},
             {"page_table": z(3, 2, dtype=torch.int32).T}, {"page_table": z(2, 0, dtype=torch.int32)}, {"page_table": z(2, 65537, dtype=torch.int32)}, {"lengths": lengths.long()},
             {"lengths": z(4, dtype=torch.int32)[::2]}, {"lengths": lengths.cpu()}, {"out": z(2, 4, 128)}, {"out": z(2, 4, 64, dtype=F16)}, {"out": z(2, 4, 128)[..., ::2]}]
    appends = [{"k": z(2, 4, 64)}, {"k": z(3, 2, 64)}, {"v": z(3, 2, 64)}, {"v": z(2, 1, 64)}, {"starts": z(2, dtype=torch.int32)}, {"starts": starts.long()}, {"cos": None},
               {"cos": None, "sin": None}, {"cos": cos.double()}, {"cos": z(50, 64, dtype=torch.float32), "sin": z(50, 64, dtype=torch.float32)}, {"sin": z(49, 32, dtype=torch.float32)},
               {"starts": None, "page_table": z(1, 3, dtype=torch.int32), "lengths": z(1, dtype=torch.int32)}, {"q": None, "out": z(2, 4, 64)}, {"k": k.clone().requires_grad_()}]
    for fn, base, changes in ((ops.paged_decode_attention, good, reads + [{"sm_scale": -1.0}, {"sm_scale": float("inf")}]),
                              (ops.paged_sparse_decode_attention, {**good, "n_pages": 2}, reads + [{"n_pages": 1}, {"n_last": 0}, {"n_first": -1}, {"n_pages": 65537}]),
                              (ops.append_to_pages, more, reads + appends)):
        fn(**base)
        for change in changes:
            with pytest.raises(_hip.AnchorAttnHipError):
                fn(**{**base, **change})
        with torch.no_grad():
            fn(**{**base, "q": z(2, 4, 64).requires_grad_()})
    with pytest.raises(_hip.AnchorAttnHipError, match="with bounds"):
        ops.paged_sparse_decode_attention(ops.PagedCache(cache.keys, cache.values), q, table, lengths, 2)
    with pytest.raises(_hip.AnchorAttnHipError, match="same memory"):
        ops.paged_decode_attention(cache, q, table, lengths, out=z(1, 4, 64).expand(2, 4, 64))
    with pytest.raises(AttributeError, match="does not change"):
        cache.keys = cache.values
    for other in (copy.copy(cache), copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert type(other) is ops.PagedCache and torch.equal(ops.paged_decode_attention(other, q, table, lengths), ops.paged_decode_attention(cache, q, table, lengths))
    assert copy.deepcopy(cache).keys.data_ptr() != cache.keys.data_ptr()
    with pytest.raises(_hip.AnchorAttnHipError, match="traced"):
        torch.func.vmap(lambda x: ops.paged_decode_attention(cache, x, table, lengths))(q[None])
    # nothing to do is no error
    none = z(0, dtype=torch.int32)
    assert ops.paged_decode_attention(cache, q[:0], table[:0], none).shape == (0, 4, 64)
    assert ops.paged_sparse_decode_attention(cache, q[:0], table[:0], none, 2)[1].shape == (0, 2, 2)
    assert ops.append_to_pages(cache, q[:0], k[:0], v[:0], cos, cos, table, lengths, starts).shape == (0, 4, 64)
    torch.cuda.synchronize()


def test_scratch_sizes():
    from anchor_attn.src.ops import _hip
    lib = _hip.lib()
    assert lib.aa_paged_sparse_workspace_bytes(0, 8, 2, 128, 16, 8, 4) == 0
    assert lib.aa_paged_sparse_workspace_bytes(2, 8, 2, 128, 16, 8, 4) >= 2 * 2 * (8 + 4) * 4
    assert isinstance(lib.aa_paged_decode_workspace_bytes(2, 8, 2, 128, 16, 8), int) and ctypes.sizeof(ctypes.c_size_t) == 8


# ---- choices that a float32 sum leaves open --------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,n_there,n_pages", [(64, 16, 300, 40), (128, 16, 700, 65), (128, 64, 1500, 100), (64, 16, 9000, 333)])
def test_scores_that_differ_by_less_than_a_float32_sum_shows(d, page, n_there, n_pages, dtype):
    """Large products of both signs that cancel and small ones that decide: neighbouring ranks differ by 2^-20 of the magnitudes and less; some are equal."""
    s = _Setup([page * n_there - 3, page * 9], 2, d, page, dtype, n_there)
    g = torch.Generator(device="cuda").manual_seed(n_there + d)
    q = s.queries(6)
    q[:, :, 0], q[:, :, 1], q[:, :, 2:] = 64.0, 64.0, q[:, :, 2:] * 2.0 ** -9
    big = (torch.randint(0, 64, s.cache.bounds[:, :, :, 0].shape, generator=g, device="cuda").float() + 64.0)[:, :, :1]
    s.cache.bounds[..., 0], s.cache.bounds[..., 1] = big.to(dtype), -big.to(dtype)
    few = torch.randint(0, 40, (s.cache.n_pages, 1), generator=g, device="cuda").expand(-1, 2)  # (40 kinds of pages)
    kinds = torch.randn(40, 2, d - 2, generator=g, device="cuda").to(dtype)
    if n_there > 500:
        s.cache.bounds[..., 2:] = s.cache.bounds[..., 2:].nan_to_num(0.25)
    else:
        s.cache.bounds[..., 2:] = kinds[few[:, :1]].expand(-1, 2, -1, -1)
    for n in (3, n_pages, n_pages + 1, 270):
        if n <= n_there:
            assert torch.equal(_ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n, 1, 1)[1], _chosen(q, s, n, 1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(BF16, 1e-38), (F16, 1e-7), (F16, 2e-5), (BF16, 1e30), (F16, 3e4)])
def test_scores_of_very_small_and_very_large_bounds(dtype, size):
    s = _Setup([16 * 400], 2, 64, 16, dtype, 5)
    s.cache.bounds.copy_((torch.randn(s.cache.bounds.shape, generator=s.g, device="cuda") * size).clamp(-6e4 if dtype == F16 else -3e38, 6e4 if dtype == F16 else 3e38).to(dtype))
    s.cache.bounds[::3] = 0
    for scale in (1.0, 1e-4, 1e4):
        q = (s.queries(4).float() * scale).to(dtype)
        for n in (3, 60, 350):
            assert torch.equal(_ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n, 1, 1)[1], _chosen(q, s, n, 1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_tables_so_wide_that_places_need_64_bits(d):
    """2100 sequences, 16 KV heads, tables for a million keys: the same bits as with tables that are as wide as they need be."""
    g = torch.Generator().manual_seed(d)
    s = _Setup([int(x) for x in torch.randint(0, 40, (2098,), generator=g)] + [3001, 900], 16, d, 256, BF16, 7)
    q = s.queries(16)
    wide = torch.full((2100, 4096), -1, dtype=torch.int32, device="cuda")
    wide[:, :s.table.shape[1]] = s.table
    assert torch.equal(_ops().paged_decode_attention(s.cache, q, wide, s.lengths), _ops().paged_decode_attention(s.cache, q, s.table, s.lengths))
    for a, b in zip(_ops().paged_sparse_decode_attention(s.cache, q, wide, s.lengths, 3), _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 3)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_longest_sequences():
    """A million keys in pages of 16: some pages chosen, nearly all, all; and of equal scores the first."""
    ops = _ops()
    s = _Setup([1 << 20, (1 << 20) - 39], 1, 64, 16, F16, 12)
    q = s.queries(3, 1.0)
    _close(ops.paged_decode_attention(s.cache, q, s.table, s.lengths), q, s, 64 ** -0.5)
    for n_pages in (100, 40000, 65535, 65536):
        out, pages = ops.paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n_pages, 1, 2)
        assert torch.equal(pages, _chosen(q, s, n_pages, 1, 2))
        _close(out, q, s, 64 ** -0.5, pages)
    s.cache.bounds.fill_(1.0)
    pages = ops.paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 50000, 1, 2)[1].cpu()
    for b, there in enumerate((65536, 65534)):
        assert pages[b, 0].tolist() == list(range(49998)) + [there - 2, there - 1]


@pytest.mark.gpu
def test_pages_that_sequences_share():
    """One prefix in several rows of the table, and a page twice in one row."""
    ops = _ops()
    s = _Setup([300, 290, 100], 2, 128, 16, BF16, 13)
    s.table[1, :12] = s.table[0, :12]
    s.table[2, 3] = s.table[2, 1]
    q = s.queries(8)
    _close(ops.paged_decode_attention(s.cache, q, s.table, s.lengths), q, s, 128 ** -0.5)
    out, pages = ops.paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 6, 1, 1)
    assert torch.equal(pages, _chosen(q, s, 6, 1, 1))
    _close(out, q, s, 128 ** -0.5, pages)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("there", [60, 1400])
def test_scores_of_zero_queries_and_infinite_bounds(there, dtype):
    """Either zero takes the larger bound, and only that one: an infinity or NaN in the other does not count."""
    s = _Setup([16 * there], 2, 64, 16, dtype, 14)
    q = s.queries(70)  # (more heads than LDS has room for, where there are many pages)
    q[:, :, 3], q[:, ::2, 4], q[:, 1::2, 4], q[0, 5, 7] = 0.0, -0.0, 0.0, float("nan")
    for pages, channel, lo, hi in ((3, 3, float("-inf"), 1.0), (5, 4, float("-inf"), 1.0), (7, 4, float("nan"), 1.0), (9, 4, -1.0, float("inf")), (11, 9, float("-inf"), float("inf"))):
        at = s.table[0, pages::13].long()
        s.cache.bounds[at, 1, 0, channel], s.cache.bounds[at, 1, 1, channel] = lo, hi
    pages = _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 20, 1, 1)[1]
    assert torch.equal(pages, _chosen(q, s, 20, 1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,hq,hkv,d,n_pages", [([3000, 40], 34, 2, 128, 20), ([16 * 25000, 7], 2, 1, 64, 300)])
def test_captured_steps_that_take_much_lds(lengths, hq, hkv, d, n_pages):
    """Sixteen columns of 128, and the scores of 25000 pages; replayed with other queries and lengths between eager steps."""
    ops = _ops()
    s = _Setup(lengths, hkv, d, 16, BF16, 15)
    q = s.queries(hq)
    step = lambda: (ops.paged_decode_attention(s.cache, q, s.table, s.lengths), *ops.paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n_pages))  # noqa: E731
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for shorter in (0, 500, 1000, 0):
        q.copy_(s.queries(hq))
        s.lengths[0] = lengths[0] - shorter
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- the edges of what may be given ------------------------------------------------------------------------------------

def _same(x, y):
    """Equal, infinities among them, and NaN in the same places."""
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.masked_fill(x.isnan(), 9.0), y.masked_fill(y.isnan(), 9.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("before,new,hkv,d,page,missing", [([3, 16], [5, 4], 2, 64, 16, 3), ([7, 0], [70, 9], 1, 128, 32, 1), ([200], [3], 2, 128, 256, 40), ([5, 1], [300, 0], 3, 64, 64, 2000)])
def test_starts_before_the_first_token(before, new, hkv, d, page, missing, dtype):
    """The rows of a larger batch from its `missing`-th token on: tokens 0 onwards have the same places as if the first sequence began with them, keys and bounds as well as
    queries and values."""
    ops, results = _ops(), []
    for first in (0, -missing):
        s = _Setup(before, hkv, d, page, dtype, 41, room=max(new))
        q, k, v = (torch.randn(sum(new), h, d, generator=s.g, device="cuda").to(dtype) for h in (2 * hkv, hkv, hkv))
        starts = torch.tensor([first, *(sum(new[:b + 1]) for b in range(len(new)))], dtype=torch.int32, device="cuda")
        lengths = torch.tensor([a + b for a, b in zip(before, new)], dtype=torch.int32, device="cuda")
        out = ops.append_to_pages(s.cache, q, k, v, *_tables(max(before) + max(new), d), s.table, lengths, starts, out=torch.full_like(q, 7.0))
        results.append((out, s.cache.keys, s.cache.values, s.cache.bounds))
    assert all(_same(a, b) for a, b in zip(*results))
    # (and they are stored: a key of every new token)
    assert int((~results[1][1].isnan()).sum()) == (sum(before) + sum(new)) * hkv * d


@pytest.mark.gpu
@pytest.mark.parametrize("size,scale", [(1e30, 1e9), (1e19, 1e19), (2e37, 5.0), (3e38, 1e38), (1e-25, 1e-19), (1e-30, 1e-10), (1e-38, 1e-38), (1e-20, 1e-19)])
@pytest.mark.parametrize("there,d", [(60, 64), (700, 64), (400, 128)])
def test_scores_whose_products_leave_float32(there, d, size, scale):
    """bf16 products beyond 2^128 or below 2^-126: the score is their float64 sum, rounded to float32 (often an infinity of its sign, or 0)."""
    s = _Setup([16 * there], 2, d, 16, BF16, there + d)
    s.cache.bounds.copy_((torch.randn(s.cache.bounds.shape, generator=s.g, device="cuda").double() * size).clamp(-3e38, 3e38).to(BF16))
    s.cache.bounds[::5] *= 0.03125
    q = (s.queries(6, 1.0).double() * scale).clamp(-3e38, 3e38).to(BF16)
    for n in (3, 20, 50):
        assert torch.equal(_ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, n, 1, 1)[1], _chosen(q, s, n, 1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("there", [60, 3000])
def test_a_score_whose_large_products_cancel(there):
    """(2^64, 2^64, 1) . (2^64, -2^64, x) is x: what two large products leave is known, not infinite."""
    s = _Setup([16 * there], 1, 64, 16, BF16, there)
    q = torch.zeros(1, 3, 64, dtype=BF16, device="cuda")
    q[..., :2], q[..., 2] = 2.0 ** 64, 1.0
    s.cache.bounds.zero_()
    s.cache.bounds[..., 0], s.cache.bounds[..., 1] = 2.0 ** 64, -2.0 ** 64
    s.cache.bounds[:, :, :, 2] = torch.randn(s.cache.n_pages, 1, 2, generator=s.g, device="cuda").to(BF16)
    s.cache.bounds[::2, :, :, :2] = 0
    assert torch.equal(_ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 20, 1, 1)[1], _chosen(q, s, 20, 1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,d", [([1, 40, 0, 17], 64), ([700, 5000, 33, 0], 128), ([20001, 3], 64)])
def test_decode_where_every_score_is_minus_infinity(lengths, d, dtype):
    """The soft-max of such scores is NaN (0 / 0), in one tile, in several and where a unit's parts are joined; other heads stay as they are, and a sequence of no keys
    gives zeros."""
    s = _Setup(lengths, 2, d, 16, dtype, 17)
    q = s.queries(4, 0.5)
    q[:, :, 0] = 1.0
    want = [_ops().paged_decode_attention(s.cache, q, s.table, s.lengths), _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 40)[0]]
    s.cache.keys[:, 0, :, 0] = float("-inf")
    s.cache.bounds[:, 0, :, 0] = float("-inf")
    got = [_ops().paged_decode_attention(s.cache, q, s.table, s.lengths), _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 40)[0]]
    for x, y in zip(got, want):
        for b, n in enumerate(lengths):
            assert bool(x[b, :2].isnan().all()) if n else bool((x[b] == 0).all())
        assert torch.equal(x[:, 2:], y[:, 2:])
    # one key that is seen is enough
    for b, n in enumerate(lengths):
        if n:
            s.cache.keys[s.table[b, (n - 1) // 16].long(), 0, (n - 1) % 16, 0] = 0.0
    got = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths)
    for b, n in enumerate(lengths):
        if n:
            assert torch.equal(got[b, :2], s.cache.values[s.table[b, (n - 1) // 16].long(), 0, (n - 1) % 16].expand(2, d))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 0, False, -0.0, float("nan"), 1e31])
def test_a_scale_that_is_given_is_not_the_default(scale):
    from anchor_attn.src.ops import _hip
    s = _Setup([40], 2, 64, 16, BF16, 18)
    q = s.queries(4)
    with pytest.raises(_hip.AnchorAttnHipError, match="sm_scale must be positive"):
        _ops().paged_decode_attention(s.cache, q, s.table, s.lengths, sm_scale=scale)
    with pytest.raises(_hip.AnchorAttnHipError, match="sm_scale must be positive"):
        _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 2, sm_scale=scale)
    assert torch.equal(_ops().paged_decode_attention(s.cache, q, s.table, s.lengths, sm_scale=None), _ops().paged_decode_attention(s.cache, q, s.table, s.lengths, sm_scale=0.125))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["keys", "values", "bounds"])
def test_a_cache_whose_tensors_get_other_memory_is_refused(name):
    """... before anything is launched: its address is the old one's."""
    from anchor_attn.src.ops import _hip
    ops = _ops()
    s = _Setup([40, 3], 2, 64, 16, BF16, 19, room=20)
    q, k, v = (torch.randn(2, h, 64, generator=s.g, device="cuda").to(BF16) for h in (4, 2, 2))
    cos, sin = _tables(100, 64)
    calls = [lambda: ops.paged_decode_attention(s.cache, q, s.table, s.lengths), lambda: ops.paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 2)[0],
             lambda: ops.append_to_pages(s.cache, q, k, v, cos, sin, s.table, s.lengths)]
    calls[2]()  # (the same once more changes nothing)
    want = [call().clone() for call in calls]
    tensor = getattr(s.cache, name)
    old, kept = tensor.data, [x.clone() for x in (s.cache.keys, s.cache.values, s.cache.bounds)]
    for other in (torch.zeros_like(old), torch.zeros_like(old[:1])):
        tensor.data = other
        for call in calls:
            with pytest.raises(_hip.AnchorAttnHipError, match="other memory"):
                call()
    tensor.data = old
    # a resize_ that moves it (to a tensor of its own first, so that the others' memory is not one with it)
    moved = [x.clone() for x in (s.cache.keys, s.cache.values, s.cache.bounds)]
    cache = ops.PagedCache(*moved)
    getattr(cache, name).resize_(4096, *old.shape[1:])
    with pytest.raises(_hip.AnchorAttnHipError, match="other memory"):
        ops.paged_decode_attention(cache, q, s.table, s.lengths)
    torch.cuda.synchronize()
    # the cache itself is as it was, and its contents may change
    assert all(_same(x, y) for x, y in zip((s.cache.keys, s.cache.values, s.cache.bounds), kept))
    for call, x in zip(calls, want):
        assert torch.equal(call(), x)
    s.cache.values.copy_(2 * s.cache.values)
    assert torch.equal(calls[0](), 2 * want[0])


@pytest.mark.gpu
def test_memory_that_is_shared_is_not_written():
    """A cache whose rows overlap without a stride of 0, or whose tensors do, is read and not appended to; outputs whose rows overlap are refused."""
    from anchor_attn.src.ops import _hip
    ops = _ops()
    z = lambda *shape: torch.zeros(shape, dtype=BF16, device="cuda")  # noqa: E731
    pool, other = torch.randn(1 << 16, device="cuda").to(BF16), torch.randn(5, 2, 16, 64, device="cuda").to(BF16)
    dense = (2 * 16 * 64, 16 * 64, 64, 1)
    at = lambda begin, strides: pool.as_strided((5, 2, 16, 64), strides, begin)  # noqa: E731
    table, lengths = torch.tensor([[3, 1], [0, 2], [4, 4]], dtype=torch.int32, device="cuda"), torch.tensor([20, 32, 17], dtype=torch.int32, device="cuda")
    q, k, starts = torch.randn(3, 4, 64, device="cuda").to(BF16), z(3, 2, 64), torch.arange(4, dtype=torch.int32, device="cuda")
    caches = []
    for strides in ((1024, 1024, 64, 1), (2048, 512, 64, 1), (8, 1024, 64, 1), (2040, 1024, 64, 1), (1024, 64, 64, 1), (64, 1024, 64, 1)):
        caches += [(at(0, strides), other, None), (other, at(0, strides), None)]
    caches += [(other, other, None), (at(0, dense), at(0, dense), None), (at(0, dense), at(9 * 1024, dense), None), (at(9 * 1024, dense), at(0, dense), None),
               (at(0, dense), at(10240 - 8, dense), None), (at(0, (4096, 1024, 64, 1)), at(2040, (4096, 1024, 64, 1)), None),
               (at(0, (4096, 1024, 64, 1)), at(1024, (4096, 1024, 64, 1)), None), (at(0, (4096, 1024, 64, 1)), at(2048, (4096, 2048, 64, 1)), None),
               (at(0, dense), other, pool[8192:8192 + 5 * 256].view(5, 2, 2, 64)), (other, at(512, dense), pool[:1280].view(5, 2, 2, 64))]
    for keys, values, bounds in caches:
        cache = ops.PagedCache(keys, values, bounds)
        before = pool.clone()
        for given in (starts, None):
            with pytest.raises(_hip.AnchorAttnHipError, match="cannot be appended to"):
                ops.append_to_pages(cache, None, k, k, None, None, table, lengths, given)
        apart = ops.PagedCache(keys.clone().contiguous(), values.clone().contiguous(), None if bounds is None else bounds.clone())
        assert torch.equal(ops.paged_decode_attention(cache, q, table, lengths), ops.paged_decode_attention(apart, q, table, lengths))
        assert torch.equal(pool, before)
    cache = ops.PagedCache(z(5, 2, 16, 64), z(5, 2, 16, 64))
    ops.append_to_pages(cache, None, k, k, None, None, table, lengths, starts)
    for strides in ((64, 64, 1), (8, 256, 1), (256, 8, 1), (128, 64, 1), (248, 64, 1), (64, 128, 1), (64, 184, 1)):
        with pytest.raises(_hip.AnchorAttnHipError, match="same memory"):
            ops.paged_decode_attention(cache, q, table, lengths, out=pool.as_strided((3, 4, 64), strides))
    for strides in ((256, 64, 1), (64, 192, 1), (1024, 72, 1), (72, 1024, 1)):
        out = pool.as_strided((3, 4, 64), strides)
        assert ops.paged_decode_attention(cache, q, table, lengths, out=out) is out


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["pages of both", "rows of both", "heads of both", "one after the other", "heads and rows"])
def test_keys_and_values_that_lie_between_each_other(layout):
    """Parts of one tensor: the same bits as from two."""
    ops, n, h, page, d = _ops(), 30, 2, 16, 64
    if layout == "pages of both":
        keys, values = torch.zeros(n, 2, h, page, d, dtype=BF16, device="cuda").unbind(1)
    elif layout == "rows of both":
        keys, values = torch.zeros(n, h, page, 2 * d, dtype=BF16, device="cuda").split(d, -1)
    elif layout == "heads of both":
        keys, values = (x.transpose(1, 2) for x in torch.zeros(n, page, 2 * h, d, dtype=BF16, device="cuda").split(h, 2))
    elif layout == "one after the other":
        keys, values = torch.zeros(2, n, h, page, d, dtype=BF16, device="cuda").unbind(0)
    else:
        both = torch.zeros(n, 2 * h * page * d, dtype=BF16, device="cuda")
        keys, values = both[:, :h * page * d].view(n, h, page, d), both[:, h * page * d:].view(n, page, h, d).transpose(1, 2)
    s = _Setup([0, 0], h, d, page, BF16, 23, room=200)
    assert s.cache.n_pages <= n
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([200, 37], [0, 200, 237]))
    q, k, v = (torch.randn(237, x, d, generator=s.g, device="cuda").to(BF16) for x in (4, h, h))
    results = []
    for cache in (s.cache, ops.PagedCache(keys, values, torch.zeros(n, h, 2, d, dtype=BF16, device="cuda"))):
        rotated = ops.append_to_pages(cache, q, k, v, *_tables(200, d), s.table, lengths, starts)
        results.append((rotated, ops.paged_decode_attention(cache, rotated[:2], s.table, lengths), *ops.paged_sparse_decode_attention(cache, rotated[:2], s.table, lengths, 5)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_tensors_that_are_told_apart_share_no_place():
    """... against all places of small tensors with strides of any kind."""
    import itertools
    import random
    ops, r = _ops(), random.Random(3)
    places = lambda dims, begin: [begin + sum(i * s for i, (s, _) in zip(at, dims)) for at in itertools.product(*(range(n) for _, n in dims))]  # noqa: E731
    told, refused = 0, 0
    for _ in range(20000):
        a, b = (sorted(((r.choice([1, 2, 3, 4, 6, 8, 12, 24]), r.randint(2, 4)) for _ in range(r.randint(0, 3))), reverse=True) for _ in range(2))
        b = r.choice([a, b])
        of_a = set(places(a, 0))
        alone = len(of_a) == len(places(a, 0))
        assert alone or not ops._own_places(a)
        if ops._own_places(a) and ops._own_places(b):
            distance = r.randint(-30, 30)
            if ops._apart(a, b, distance):
                told += 1
                assert not of_a & set(places(b, distance))
            else:
                refused += bool(of_a & set(places(b, distance)))
    assert told > 1000 and refused > 1000


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_what_is_no_tensor_or_whole_number_is_refused(grad):
    """By the error that every refused call raises, with gradients recorded or not."""
    import numpy as np
    from anchor_attn.src.ops import _hip
    ops = _ops()
    s = _Setup([40, 3], 2, 64, 16, BF16, 24, room=20)
    q, k = s.queries(4), torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    cos, sin = _tables(100, 64)
    steps = {"cache": s.cache, "q": q, "page_table": s.table, "lengths": s.lengths}
    for fn, given, names in ((ops.paged_decode_attention, steps, ("q", "page_table", "lengths", "out")),
                             (ops.paged_sparse_decode_attention, {**steps, "n_pages": 2}, ("q", "page_table", "lengths", "out")),
                             (ops.append_to_pages, {**steps, "k": k, "v": k, "cos": cos, "sin": sin}, ("q", "k", "v", "cos", "sin", "page_table", "lengths", "starts", "out"))):
        for name in names:
            for other in ([1.0], "x", 3, np.zeros((2, 4, 64), np.float32)):
                with torch.set_grad_enabled(grad), pytest.raises(_hip.AnchorAttnHipError):
                    fn(**{**given, name: other})
    for change in ({"n_pages": 2.5}, {"n_pages": "2"}, {"n_pages": float("inf")}, {"n_first": float("nan")}, {"n_pages": None}, {"n_first": 0.5}, {"n_last": 1.5}, {"n_last": None}):
        with pytest.raises(_hip.AnchorAttnHipError, match="whole numbers"):
            ops.paged_sparse_decode_attention(**{**steps, "n_pages": 3, **change})
    want = ops.paged_sparse_decode_attention(**steps, n_pages=2)
    assert all(torch.equal(a, b) for a, b in zip(want, ops.paged_sparse_decode_attention(**steps, n_pages=np.int64(2), n_first=torch.tensor(1), n_last=1.0)))


@pytest.mark.parametrize("fn", ["aa_paged_decode_fwd", "aa_paged_sparse_decode_fwd"])
@pytest.mark.parametrize("scale", [3e38, 2.5e38, -1.0, float("-inf")])
def test_scales_that_leave_float32_are_refused(fn, scale):
    """The kernels multiply scores by sm_scale * log2 e: an infinity there gives NaN for the largest score."""
    from anchor_attn.src.ops import _hip
    struct = _hip.PagedCacheStruct(*CACHE.values())
    with pytest.raises(_hip.AnchorAttnHipError, match="sm_scale"):
        _hip.check(getattr(_hip.lib(), fn)(ctypes.addressof(struct), _hip.PAGED_STEP.pack(*{**STEP, "sm_scale": scale}.values()), None))


# ---- what the documents allow -----------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_bounds_tell_infinities_from_the_largest_numbers(dtype):
    """Infinite keys give infinite bounds, the largest finite ones finite bounds, in the page's first append and in one that widens them; NaN of either sign both."""
    ops = _ops()
    s = _Setup([0], 1, 64, 16, dtype, 25, room=40)
    most = torch.finfo(dtype).max
    k = torch.randn(40, 1, 64, generator=s.g, device="cuda").to(dtype)
    for row in (2, 17, 30):
        for channel, x in enumerate((float("inf"), float("-inf"), most, -most, float("nan"), -float("nan"), -0.0)):
            k[row + channel % 3, 0, channel] = x
            k[row + (channel + 1) % 3, 0, 32 + channel] = x
        k[row, 0, 20], k[row + 1, 0, 20] = float("inf"), float("-inf")
        k[row, 0, 21], k[row + 1, 0, 21] = float("inf"), float("nan")
        k[row, 0, 22], k[row + 1, 0, 22] = most, float("inf")
    for lo, hi in ((0, 3), (3, 16), (16, 19), (19, 40)):
        ops.append_to_pages(s.cache, None, k[lo:hi], k[lo:hi], None, None, s.table, torch.tensor([hi], dtype=torch.int32, device="cuda"),
                            torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda"))
        for i in range(0, hi, 16):
            page, rows = int(s.table[0, i // 16]), k[i:min(hi, i + 16), 0]
            assert _same(s.cache.keys[page, 0, :rows.shape[0]], rows) and _same(s.cache.values[page, 0, :rows.shape[0]], rows)
            assert _same(s.cache.bounds[page, 0], torch.stack((rows.amin(0), rows.amax(0))))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,hq,hkv,d,page", [(1, 14, 2, 64, 16), (97, 32, 8, 128, 64), (300, 4, 1, 128, 256)])
def test_append_one_token_each_in_fp16(batch, hq, hkv, d, page):
    _append_and_check([(37 * b) % 211 for b in range(batch)], [1] * batch, hq, hkv, d, page, F16, "heads", steps=True, seed=batch)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_that_lie_as_far_apart_as_they_may(dtype):
    """Rows 16384 elements apart, appended to and read: the same bits as from dense pages."""
    ops, n, h, page, d = _ops(), 11, 3, 32, 128
    far = [torch.full((n, page, 16384), float("nan"), dtype=dtype, device="cuda")[:, :, 128:128 + h * 256].unflatten(2, (h, 256))[..., 64:64 + d].transpose(1, 2) for _ in range(2)]
    s = _Setup([0, 0], h, d, page, dtype, 26, room=100)
    assert s.cache.n_pages <= n and far[0].stride()[2] == 16384
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([97, 31], [0, 97, 128]))
    q, k, v = (torch.randn(128, x, d, generator=s.g, device="cuda").to(dtype) for x in (2 * h, h, h))
    results = []
    for cache in (s.cache, ops.PagedCache(*far, torch.zeros(n, h, 2, d, dtype=dtype, device="cuda"))):
        rotated = ops.append_to_pages(cache, q, k, v, *_tables(100, d), s.table, lengths, starts)
        results.append((rotated, ops.paged_decode_attention(cache, rotated[:2], s.table, lengths), *ops.paged_sparse_decode_attention(cache, rotated[:2], s.table, lengths, 3)))
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool(results[1][1].isfinite().all())


@pytest.mark.gpu
def test_views_that_repeat_or_leave_out():
    """Expanded queries, one row of a table for all sequences, a table that is part of a wider one, lengths from the middle of a tensor."""
    ops = _ops()
    s = _Setup([300, 270, 5], 2, 64, 16, BF16, 27)
    q = s.queries(4)
    run = lambda q, t, n: (ops.paged_decode_attention(s.cache, q, t, n), *ops.paged_sparse_decode_attention(s.cache, q, t, n, 6))  # noqa: E731
    want = run(q, s.table, s.lengths)
    wide, more = torch.full((3, 100), -1, dtype=torch.int32, device="cuda"), torch.tensor([9, 9, 300, 270, 5, 9], dtype=torch.int32, device="cuda")
    wide[:, 3:3 + s.table.shape[1]] = s.table
    assert all(torch.equal(a, b) for a, b in zip(run(q, wide[:, 3:3 + s.table.shape[1]], more[2:5]), want))
    lengths = torch.tensor([300, 100, 0], dtype=torch.int32, device="cuda")
    one = run(q[:1].expand(3, 4, 64).contiguous(), s.table[:1].repeat(3, 1), lengths)
    assert all(torch.equal(a, b) for a, b in zip(run(q[:1].expand(3, 4, 64), s.table[:1].expand(3, -1), lengths), one))
    one_head = run(q[:, :1].expand(3, 4, 64).contiguous(), s.table, s.lengths)
    assert all(torch.equal(a, b) for a, b in zip(run(q[:, :1].expand(3, 4, 64), s.table, s.lengths), one_head))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(4096, 1, 64), (3000, 1500, 64), (9000, 9000, 64), (640, 20, 128)])
def test_many_heads(hq, hkv, d):
    s = _Setup([70, 33], hkv, d, 16, BF16, 28)
    q = s.queries(hq, 1.0)
    out, (sparse, pages) = _ops().paged_decode_attention(s.cache, q, s.table, s.lengths), _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 4)
    for b, n in enumerate(s.host):
        there = (n + 15) // 16
        at = s.table[b, :there].long()
        k, v = (x[at].transpose(0, 1).flatten(1, 2)[:, :n].double() for x in (s.cache.keys, s.cache.values))
        x = q[b].view(hkv, hq // hkv, d).double()
        score = (x @ k.transpose(1, 2)) * d ** -0.5
        lo, hi = (s.cache.bounds[at, :, i].transpose(0, 1).double() for i in (0, 1))
        page_score = (x.clamp(min=0) @ hi.transpose(1, 2) + x.clamp(max=0) @ lo.transpose(1, 2)).amax(1).float()
        chosen = torch.zeros(hkv, there, dtype=torch.bool, device="cuda")
        if there <= 4:
            chosen[:] = True
        else:  # (five pages: the first, the last and two between are read)
            page_score[:, 0] = page_score[:, -1] = float("inf")
            chosen.scatter_(1, page_score.sort(dim=1, descending=True, stable=True).indices[:, :4], True)
        assert torch.equal(chosen, torch.zeros(hkv, there + 1, dtype=torch.bool, device="cuda").scatter_(1, pages[b].long() % (there + 1), True)[:, :there])
        hidden = ~chosen.repeat_interleave(16, 1)[:, None, :n]
        for got, p in ((out, score.softmax(-1)), (sparse, score.masked_fill(hidden, float("-inf")).softmax(-1))):
            want = (p @ v).reshape(hq, d)
            relative = 2.0 * d * 2.0 ** -24 * float((x.abs() @ k.abs().transpose(1, 2)).amax()) * d ** -0.5 + 2.0 ** -14 + U[BF16] ** 2 + n * 2.0 ** -24
            bound = U[BF16] * want.abs() * 1.001 + relative * (p @ v.abs()).reshape(hq, d) + 2.0 ** -25
            assert bool(((got[b].double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_the_most_sequences():
    """65535 of them, of 0 to 16 keys: a sequence's output is the same as that of a batch of its own."""
    ops, n = _ops(), 65535
    g = torch.Generator(device="cuda").manual_seed(29)
    cache = ops.PagedCache.empty(4096, 1, 16, 64)
    cache.keys.normal_(generator=g), cache.values.normal_(generator=g)
    table = torch.randint(0, 4096, (n, 1), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.randint(0, 17, (n,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn(n, 2, 64, generator=g, device="cuda").to(BF16)
    out = ops.paged_decode_attention(cache, q, table, lengths)
    for b in (0, 1, 63, 64, 255, 256, 257, 32768, 65279, 65280, 65533, 65534):
        assert torch.equal(out[b:b + 1], ops.paged_decode_attention(cache, q[b:b + 1], table[b:b + 1], lengths[b:b + 1]))
    keys, values = cache.keys[table[:, 0].long(), 0], cache.values[table[:, 0].long(), 0]
    score = (q.float() @ keys.float().transpose(1, 2)) / 8
    p = score.masked_fill(torch.arange(16, device="cuda") >= lengths[:, None, None], float("-inf")).softmax(-1).nan_to_num(0.0)
    # (besides the output's rounding 2 * 64 * 2^-24 * sum |q k| / 8, below 2^-13 here, 2^-14 of exp2, 2^-16 of the pairs: 2^-12 of sum p |v|)
    assert bool(((out.float() - p @ values.float()).abs() <= 2.0 ** -8 * (p @ values.float()).abs() * 1.01 + 2.0 ** -12 * (p @ values.abs().float())).all())
    # and appended to: every sequence's next token, to pages of their own
    pool = ops.PagedCache.empty(n, 1, 16, 64)
    own = torch.randperm(n, generator=g, device="cuda").int()[:, None]
    k = torch.randn(n, 1, 64, generator=g, device="cuda").to(BF16)
    pool.keys.zero_(), pool.values.zero_()
    ops.append_to_pages(pool, None, k, q[:, :1], None, None, own, lengths)
    there = lengths > 0
    at, slot = own[there, 0].long(), lengths[there].long() - 1
    assert torch.equal(pool.keys[at, 0, slot], k[there, 0]) and torch.equal(pool.values[at, 0, slot], q[there, 0])
    assert int((pool.keys != 0).any(-1).sum()) == int(there.sum())


@pytest.mark.gpu
def test_a_prompt_of_a_million_tokens():
    ops, n, page = _ops(), (1 << 20) - 37, 64
    g = torch.Generator(device="cuda").manual_seed(30)
    cache = ops.PagedCache.empty(n // page + 1, 1, page, 64, F16)
    table = torch.randperm(cache.n_pages, generator=g, device="cuda").int()[None]
    k, v = (torch.randn(n, 1, 64, generator=g, device="cuda").to(F16) for _ in range(2))
    ops.append_to_pages(cache, None, k, v, None, None, table, torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    for pool, x in ((cache.keys, k), (cache.values, v)):
        assert torch.equal(pool[table[0].long(), 0].flatten(0, 1)[:n], x[:, 0])
    full = n // page
    assert torch.equal(cache.bounds[table[0, :full].long(), 0, 0], k[:full * page, 0].view(full, page, 64).amin(1))
    assert torch.equal(cache.bounds[table[0, :full].long(), 0, 1], k[:full * page, 0].view(full, page, 64).amax(1))
    assert torch.equal(cache.bounds[table[0, full].long(), 0], torch.stack((k[full * page:, 0].amin(0), k[full * page:, 0].amax(0))))


@pytest.mark.gpu
def test_inference_mode_and_threads():
    import threading
    ops = _ops()
    s = _Setup([3000, 5000, 100], 4, 128, 64, BF16, 31, room=64)
    q = [s.queries(16) for _ in range(4)]
    step = lambda x: (ops.paged_decode_attention(s.cache, x, s.table, s.lengths), *ops.paged_sparse_decode_attention(s.cache, x, s.table, s.lengths, 9))  # noqa: E731
    want = [step(x) for x in q]
    with torch.inference_mode():
        cache = ops.PagedCache(s.cache.keys.clone(), s.cache.values.clone(), s.cache.bounds.clone())
        assert torch.equal(ops.paged_decode_attention(cache, q[0], s.table, s.lengths), want[0][0])
        k = torch.zeros(3, 4, 128, dtype=BF16, device="cuda")
        ops.append_to_pages(cache, None, k, k, None, None, s.table, s.lengths + 1)
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got[i] = [step(q[i]) for _ in range(10)]
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for outs, x in zip(got, want):
        assert all(torch.equal(a, b) for one in outs for a, b in zip(one, x))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,batch,width", [(32, 8, 128, 1, 128), (32, 8, 128, 1, 129), (32, 8, 128, 32, 230), (32, 8, 128, 32, 231), (14, 2, 64, 1, 215), (14, 2, 64, 1, 216),
                                                  (71, 1, 128, 3, 24), (71, 1, 128, 3, 25), (2, 2, 64, 1, 315), (2, 2, 64, 2, 316), (256, 256, 64, 1, 566), (256, 256, 64, 1, 567)])
def test_sparse_decode_on_both_sides_of_one_launch_or_two(hq, hkv, d, batch, width):
    """Tables of widths where scoring and choosing become two launches, with the same sequences."""
    lengths = [16 * (width if hkv < 99 else 60) - 3 - 16 * b for b in range(min(batch, 3))] + [100] * (batch - 3)
    s = _Setup(lengths, hkv, d, 16, BF16, width)
    if s.table.shape[1] < width:
        s.table = torch.cat((s.table, torch.full((batch, width - s.table.shape[1]), -1, dtype=torch.int32, device="cuda")), 1)
    assert s.table.shape[1] == width
    q = s.queries(hq)
    out, pages = _ops().paged_sparse_decode_attention(s.cache, q, s.table, s.lengths, 11, 1, 2)
    assert torch.equal(pages, _chosen(q, s, 11, 1, 2))
    _close(out, q, s, d ** -0.5, pages)
