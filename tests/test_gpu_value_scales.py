"""Attention over 8-bit pages whose values' scales lie as far apart as it is right for: every key counts in the softmax's sum, however
small its value is."""
import math

import pytest
import torch

import cache8_tools as c8
from test_gpu_cache8 import run as run_apart
from test_gpu_shared_prefix import K, case, run  # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu


def scaled(kv, how, seed=3):
    """The pages with other values: `wide`, scales spread evenly over 2^80; `zeros`, two keys in three with a value of zeros (which has
    the least scale there is) beside values of up to 2^24; `all zeros`, but for one key in 64."""
    g = torch.Generator().manual_seed(seed)
    p, two, kvh, page, d1 = kv.shape
    x = torch.randn(p, kvh, page, d1 - 1, generator=g, dtype=torch.float64)
    r = torch.rand(p, kvh, page, 1, generator=g, dtype=torch.float64)
    if how == "wide":
        x = x * 2.0 ** (80 * (r - 0.5))
    else:
        x = torch.where(r < (2 / 3 if how == "zeros" else 63 / 64), 0.0, x.clamp(-4, 4) * 2.0 ** 22)
    codes, e = c8.encode(x)
    c, s = (t.clone() for t in c8.split(kv))
    c[:, 1], s[:, 1] = codes, (e + 127).to(torch.uint8)
    return c8.pack(c, s.long() - 127)


def lost(q, kv, table, rows, scale, sinks):
    """What halves lose that are subnormal: a weight is off by 2^-25 at most, half their spacing, where the key with the largest
    score + exponent of its value's scale weighs 2^14. On the result of a head that is 2^-39 2^(that - log2 of the softmax's sum) times the
    sum of the values' |codes|. It tells where a key with a value of (nearly) zeros has more than 2^28 times the others' weight."""
    values, page, heads, kvh = c8.decode(kv), kv.shape[3], q.shape[1], kv.shape[2]
    scales = c8.split(kv)[1].double() - 127
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(rows.n_rows):
        n = int(rows.kv_len[b])
        pages = table[int(rows.row_slot[b]), :-(-n // page)].long()
        k, v = (values[pages, i].transpose(1, 2).reshape(-1, kvh, q.shape[2])[:n] for i in (0, 1))
        e = scales[pages, 1].transpose(1, 2).reshape(-1, kvh)[:n]
        codes = (v.abs() * 2.0 ** -e[..., None]).sum(0).repeat_interleave(heads // kvh, 0)
        s = torch.einsum("hd,khd->hk", q[b].double(), k.repeat_interleave(heads // kvh, 1)) * scale
        total = torch.logaddexp(s.logsumexp(-1), sinks.double()) / math.log(2)
        most = (s / math.log(2) + e.T.repeat_interleave(heads // kvh, 0)).amax(-1)
        out[b] = 2.0 ** (most - total - 39)[:, None] * codes
    return out


def within(got, want, mass, lost, halves):
    """Half a step of bfloat16 on the result, half a step of the weights' type on the sum of weight x |value|, 2^-12 for the 32-bit sums and
    the exponential's 2^-22 on exponents up to a few hundred, and what subnormal halves lose."""
    bound = 2.0 ** -8 * want.abs() + ((2.0 ** -11 if halves else 2.0 ** -8) + 2.0 ** -12) * mass * 1.01 + lost + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{(off / bound).max().item():.3g} times what rounding explains"


@pytest.mark.parametrize("sharp", [0.0, 1.5, 20.0])                   # equal weights; ordinary ones; a few keys that take nearly all
@pytest.mark.parametrize("how", ["wide", "zeros", "all zeros"])
@pytest.mark.parametrize("form", [None, (1, 0, 0), (4, 0, 1), (1, 1, 0)])
def test_values_of_very_unequal_size(K, how, sharp, form, monkeypatch):   # noqa: F811
    q, kv, table, rows, shared = case([(9, [1, 130, 64, 300])], [700, 65], 8, 2, 64, 64, True, seed=5)
    kv, q = scaled(kv, how), (q.float() * sharp / 1.5).to(q.dtype)
    sinks = torch.linspace(-2, 3, 8)
    want, mass = c8.attend(q, kv, table, rows, 0.125, 0, sinks)
    less = lost(q, kv, table, rows, 0.125, sinks)
    if form is not None:
        monkeypatch.setattr(K, "_row_splits", lambda *a: form, raising=False)
    within(run_apart(K, q, kv, table, rows, 0.125, 0, sinks), want, mass, less, halves=True)
    within(run(K, q, kv, table, rows, 0.125, sinks, shared), want, mass, less, halves=False)
