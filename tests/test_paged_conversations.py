"""Long and shared conversations in a key/value cache in pages - appending with norms and positions apart from places, decode that counts attention, eviction,
decode over a shared prefix - against plain float64 implementations, at the lengths, pages and layouts where tiles, pages and shares of the work end.

Tolerances beside those of tests/test_paged_cache.py (u: half a step of the 16-bit type).
Norm and rotation: a float32 sum of D squares is off by at most D * 2^-24 of it, its inverse root by half of that and 2^-22, three products by 2^-24 each,
the rotation by 2^-23 of its products' magnitudes: (D / 2 + 16) * 2^-24 of the magnitudes, and u of the result."""
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
