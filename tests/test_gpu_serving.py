"""The serving operators on the GPU against their 64-bit definitions (tests/serving_ref.py).

Every cache is poisoned: pages nobody owns, rows behind a sequence's length and entries behind its page
list hold NaN and ids outside the pool, so a read past the end shows. Tolerances of an attention output,
with u half a step of the output's type and vmax the largest |v|: u |ref| for the stored rounding, u vmax
for probabilities rounded to the type before they meet the values (sum of p is 1), and for fp16 half its
smallest step per key; the scores' fp32 sums may be off by hd steps of sum |q k| scale, which moves each
probability by twice that."""
import ctypes
import math

import pytest
import torch

from tests import serving_ref as R

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _pools(lens, n_kv, hd, page, dtype, g, order="pages", spare=3):
    """CPU pools [pages, page, n_kv, hd] poisoned outside the sequences' slots, and a shuffled table."""
    need = [-(-n // page) for n in lens]
    total, width = sum(need) + spare, max(1, max(need)) + 1
    perm = torch.randperm(total, generator=g)
    table = torch.full((len(lens), width), 10 ** 9, dtype=torch.int32)
    k = torch.full((total, page, n_kv, hd), NAN, dtype=dtype)
    v = torch.full_like(k, NAN)
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[at:at + need[b]].int()
        at += need[b]
        slot = torch.arange(n)
        pages = table[b].long()[slot // page]
        k[pages, slot % page] = torch.randn(n, n_kv, hd, generator=g).to(dtype)
        v[pages, slot % page] = torch.randn(n, n_kv, hd, generator=g).to(dtype)
    return k, v, table


def _cuda_pool(x, order):
    """On the GPU with heads outside slots ("heads") or the plain order ("slots")."""
    if order == "heads":
        return x.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
    return x.cuda()


def _cache(k, v, table, lens, order="heads", track=None):
    from opentars_b200 import serving as S
    length = torch.tensor(lens, dtype=torch.int32).cuda()
    more = {} if track is None else dict(weight=track[0].cuda(), pos=track[1].cuda(), seen=track[2].cuda())
    return S.PagedCache(_cuda_pool(k, order), _cuda_pool(v, order), table.cuda(), length, **more)


def _finite(x):
    return torch.nan_to_num(x.float(), 0, 0, 0).abs()


def _tolerance(ref, q, k, v, scale, dtype):
    u = torch.finfo(dtype).eps / 2
    vmax = float(_finite(v).max()) if v.numel() else 0.0
    hd = q.shape[-1]
    smax = abs(scale) * hd * float(_finite(q).max()) * float(_finite(k).max())
    slots = k.shape[0] * k.shape[1]
    tiny = slots * 2.0 ** -25 if dtype == torch.float16 else 0.0
    return u * ref.abs() + (u + tiny + 2 * hd * 2.0 ** -23 * smax / 8 + 2.0 ** -18) * vmax


def _close(got, ref, tol, what=""):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN where there is none, or none where one is"
    bad = (got - ref).abs() > tol
    bad &= ~torch.isnan(ref)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(got - ref).abs()[bad].max()}"


def _no_error():
    from opentars_b200 import serving as S
    torch.cuda.synchronize()
    assert S.device_error(clear=True) == 0


# dtype, head dim, page, kv heads, group, lengths, window, sinks, pool order
ATTEND = [
    (torch.bfloat16, 128, 16, 2, 2, [1, 0, 37, 300], 0, 0, "heads"),
    (torch.float16, 64, 32, 3, 1, [64, 65, 63, 1, 0], 0, 0, "slots"),
    (torch.bfloat16, 256, 64, 1, 4, [513, 128, 700], 512, 4, "heads"),
    (torch.float16, 128, 16, 2, 7, [1000, 17, 16, 15], 100, 1, "slots"),
    (torch.bfloat16, 64, 128, 1, 16, [257], 0, 0, "heads"),
    (torch.bfloat16, 128, 256, 1, 33, [400, 2], 64, 30, "heads"),
    (torch.float16, 256, 16, 2, 3, [130, 5], 1, 0, "slots"),
    (torch.bfloat16, 128, 32, 8, 2, [2500] + [3] * 20, 0, 0, "heads"),
    (torch.float16, 64, 16, 1, 8, [9000], 0, 0, "heads"),
    (torch.bfloat16, 128, 16, 1, 2, [4000, 90], 2 ** 31 - 1, 2 ** 31 - 1, "slots"),
    (torch.float16, 128, 64, 2, 2, [600, 700], 40, 5000, "heads"),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{c[0]}-{c[1]}-p{c[2]}-{c[3]}x{c[4]}-{max(c[5])}-w{c[6]}-s{c[7]}")
@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
def test_attend(case, weights):
    from opentars_b200 import serving as S
    dtype, hd, page, kv, G, lens, window, sinks, order = case
    g = torch.Generator().manual_seed(sum(lens) + hd)
    k, v, table = _pools(lens, kv, hd, page, dtype, g)
    q = torch.randn(len(lens), kv * G, hd, generator=g).to(dtype)
    scale = hd ** -0.5
    track = None
    cap = table.shape[1] * page + 5
    if weights:
        w0 = torch.rand(len(lens), kv, cap, generator=g)
        track = (w0, torch.zeros(len(lens), kv, cap, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32))
    cache = _cache(k, v, table, lens, order, track)
    ref, prob = R.attend(k, v, table, lens, q, scale, window, sinks, page)
    w_out = torch.full((len(lens), kv, cap), 7.0, device="cuda") if weights else None
    out = S.attend(cache, q.cuda(), scale, window=window, sinks=sinks, weight_out=w_out)
    _no_error()
    _close(out, ref, _tolerance(ref, q, k, v, scale, dtype), "out")
    if weights:
        smax = scale * hd * float(_finite(q).max()) * float(_finite(k).max())
        for b, n in enumerate(lens):
            got = w_out[b].cpu().double()
            want = w0[b, :, :n].double() + prob[b]
            tol = 2.0 ** -23 * want + prob[b] * (2 * hd * 2.0 ** -23 * smax / 8 + 2.0 ** -18) + 1e-30
            assert ((got[:, :n] - want).abs() <= tol).all(), b
            assert (got[:, n:] == 7.0).all()                     # slots behind the length are left alone
        acc = cache.weight.clone()
        S.attend(cache, q.cuda(), scale, window=window, sinks=sinks, weight_out=cache.weight)   # in place
        for b, n in enumerate(lens):
            assert torch.equal(cache.weight[b, :, :n], w_out[b, :, :n])
            assert torch.equal(cache.weight[b, :, n:], acc[b, :, n:])


def test_attend_leaves_hidden_slots_out():
    """NaN and infinities in slots that the window hides do not reach the output or the weights."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(5)
    lens, kv, hd, page, window, sinks = [333, 90], 2, 128, 16, 50, 3
    k, v, table = _pools(lens, kv, hd, page, torch.bfloat16, g)
    for b, n in enumerate(lens):
        for s in range(sinks, n - window):
            p = int(table[b, s // page])
            k[p, s % page], v[p, s % page] = (NAN, math.inf) if s % 2 else (-math.inf, NAN)
    q = torch.randn(2, 4, hd, generator=g).bfloat16()
    cap = table.shape[1] * page
    cache = _cache(k, v, table, lens, "heads", (torch.zeros(2, kv, cap), torch.zeros(2, kv, cap, dtype=torch.int32),
                                                torch.tensor(lens, dtype=torch.int32)))
    ref, prob = R.attend(k, v, table, lens, q, 0.1, window, sinks, page)
    out = S.attend(cache, q.cuda(), 0.1, window=window, sinks=sinks, weight_out=cache.weight)
    _no_error()
    _close(out, ref, _tolerance(ref, q, k[:, :, :, :], v, 0.1, torch.bfloat16))
    for b, n in enumerate(lens):
        assert (cache.weight[b, :, sinks:n - window] == 0).all()
        assert torch.isfinite(cache.weight[b]).all()


def test_attend_takes_strided_rows_and_visible_nonfinite_values():
    """q and out as slices of wider rows; a visible NaN or infinity gives what the formula gives."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(6)
    lens, kv, hd, page = [40, 40, 40, 40], 2, 64, 32
    k, v, table = _pools(lens, kv, hd, page, torch.float16, g)
    v[int(table[1, 0]), 3, 0, 5] = math.inf                    # one element of one head's value
    v[int(table[2, 0]), 3, 1, 7] = NAN
    k[int(table[3, 0]), 3, 0] = NAN                            # a whole key: every output of the head is NaN
    wide = torch.randn(4, 10, 2 * hd, generator=g).half()
    q = wide[:, 2:6, hd:]
    cache = _cache(k, v, table, lens)
    ref, _ = R.attend(k, v, table, lens, q, 0.125, 0, 0, page)
    dev = torch.zeros(4, 8, hd, dtype=torch.float16, device="cuda")
    out = S.attend(cache, wide.cuda()[:, 2:6, hd:], 0.125, out=dev[:, ::2])
    _no_error()
    assert out.data_ptr() == dev.data_ptr() and (dev[:, 1::2] == 0).all()
    assert math.isinf(float(ref[1, 0, 5])) and torch.isnan(ref[2, 2:, 7]).all() and torch.isnan(ref[3, :2]).all()
    assert torch.equal(torch.isinf(out.cpu()), torch.isinf(ref.float()))
    inf = torch.isinf(ref)
    tol = _tolerance(torch.where(inf, 0.0, ref), q, k, v, 0.125, torch.float16)
    _close(torch.where(inf.cuda(), 0.0, out.float()), torch.where(inf, 0.0, ref), tol)


# dtype, head dim, page, kv heads, group, (cached, new) per sequence, window, sinks, order
PROMPT = [
    (torch.bfloat16, 128, 16, 1, 2, [(0, 1), (0, 300), (5, 0), (77, 40)], 0, 0, "heads"),
    (torch.float16, 64, 32, 2, 1, [(0, 129), (128, 128), (1, 127)], 0, 0, "slots"),
    (torch.bfloat16, 256, 64, 1, 4, [(100, 200), (0, 70)], 64, 4, "heads"),
    (torch.float16, 256, 16, 1, 2, [(0, 150)], 0, 0, "slots"),
    (torch.float16, 128, 16, 2, 7, [(33, 50), (0, 20)], 30, 1, "slots"),
    (torch.bfloat16, 64, 128, 1, 16, [(0, 90), (1000, 3)], 0, 0, "heads"),
    (torch.bfloat16, 128, 256, 1, 3, [(300, 260)], 1, 0, "heads"),
    (torch.bfloat16, 128, 16, 2, 1, [(0, 1)] * 9, 0, 0, "heads"),
    (torch.float16, 64, 16, 1, 33, [(3, 21)], 10, 2, "slots"),
    (torch.bfloat16, 128, 64, 1, 4, [(700, 170)], 2 ** 31 - 1, 2 ** 31 - 1, "heads"),
    (torch.bfloat16, 128, 32, 1, 2, [(2000, 4), (10, 4), (0, 4)], 300, 40, "slots"),
    # few rows a sequence
    (torch.bfloat16, 128, 16, 2, 2, [(1000, 4), (3, 4), (0, 0), (0, 1), (64, 7)], 0, 0, "heads"),
    (torch.float16, 256, 64, 1, 4, [(600, 8), (0, 3)], 512, 4, "heads"),
    (torch.bfloat16, 64, 16, 3, 1, [(5, 31), (500, 33), (15, 1)], 20, 3, "slots"),
    (torch.float16, 128, 16, 1, 7, [(100, 2), (0, 5), (333, 1)], 0, 0, "heads"),
    (torch.bfloat16, 256, 16, 1, 16, [(40, 2)], 1, 0, "heads"),
    (torch.float16, 64, 256, 1, 20, [(300, 1), (0, 2)], 50, 260, "slots"),
    (torch.bfloat16, 128, 16, 1, 2, [(9000, 5)], 0, 0, "heads"),
    (torch.float16, 128, 64, 2, 3, [(1, 1)] * 40 + [(0, 60)], 0, 0, "heads"),
]


def _rows(case, extra, g):
    dtype, hd, page, kv, G, seqs, window, sinks, order = case
    cu = [0]
    for _, n in seqs:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + extra, kv * G, hd, generator=g).to(dtype)
    return q, torch.tensor(cu, dtype=torch.int32)


@pytest.mark.parametrize("case", PROMPT, ids=lambda c: f"{c[0]}-{c[1]}-p{c[2]}-{c[3]}x{c[4]}-{c[5][0]}-w{c[6]}-s{c[7]}")
def test_attend_prompt(case):
    from opentars_b200 import serving as S
    dtype, hd, page, kv, G, seqs, window, sinks, order = case
    g = torch.Generator().manual_seed(hd + len(seqs))
    lens = [c + n for c, n in seqs]
    k, v, table = _pools(lens, kv, hd, page, dtype, g)
    q, cu = _rows(case, 3, g)
    cache = _cache(k, v, table, lens, order)
    scale = hd ** -0.5
    ref = R.attend_prompt(k, v, table, lens, q, cu, scale, window, sinks, page)
    out = torch.full(q.shape, 9.0, dtype=dtype, device="cuda")
    S.attend_prompt(cache, q.cuda(), cu.cuda(), scale, window=window, sinks=sinks, out=out)
    _no_error()
    n = int(cu[-1])
    assert (out[n:] == 9.0).all()                              # rows behind the last sequence are left alone
    _close(out[:n], ref[:n], _tolerance(ref[:n], q, k, v, scale, dtype))


def test_attend_prompt_keeps_later_tokens_out():
    """NaN and infinities in a later token's key and value do not reach the rows before it."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(8)
    lens, hd, page = [200], 128, 16
    k, v, table = _pools(lens, 1, hd, page, torch.bfloat16, g)
    for s, (kk, vv) in {60: (NAN, 1.0), 90: (1.0, NAN), 91: (1.0, math.inf), 150: (-math.inf, NAN)}.items():
        k[int(table[0, s // page]), s % page] = kk
        v[int(table[0, s // page]), s % page] = vv
    q = torch.randn(200, 2, hd, generator=g).bfloat16()
    cu = torch.tensor([0, 200], dtype=torch.int32)
    ref = R.attend_prompt(k, v, table, lens, q, cu, 0.09, 20, 0, page)
    out = S.attend_prompt(_cache(k, v, table, lens), q.cuda(), cu.cuda(), 0.09, window=20)
    _no_error()
    assert torch.isfinite(ref[:60]).all() and torch.isfinite(ref[80:90]).all() and torch.isfinite(ref[170:]).all()
    assert torch.isnan(ref[60]).all()
    _close(out, ref, _tolerance(ref, q, k, v, 0.09, torch.bfloat16))


@pytest.mark.parametrize("n", [9, 300])
def test_attend_prompt_rows_at_negative_positions_get_zeros(n):
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(9)
    k, v, table = _pools([5], 1, 64, 16, torch.bfloat16, g)
    q = torch.randn(n, 1, 64, generator=g).bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int32)
    out = S.attend_prompt(_cache(k, v, table, [5]), q.cuda(), cu.cuda(), 0.125)
    _no_error()
    assert (out[:n - 5] == 0).all() and (out[n - 5:] != 0).any()
    ref = R.attend_prompt(k, v, table, [5], q, cu, 0.125, 0, 0, 16)
    _close(out, ref, _tolerance(ref, q, k, v, 0.125, torch.bfloat16))


@pytest.mark.parametrize("op,n,room", [("attend", 1, 0), ("prompt", 1, 0), ("prompt", 1, 600), ("prompt", 50, 0)])
def test_bad_pages_and_lengths_are_left_out_and_recorded(op, n, room):
    """Ids outside the pool inside the used slots, and a length beyond the page list: the kernels check
    every id against the pool and clamp the length before they read. (Room in the page list for many more
    slots takes a chunk of few rows to the kernel that splits the length.)"""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(10)
    lens, hd, page = [100, 70, 64], 128, 16
    k, v, table = _pools(lens, 2, hd, page, torch.bfloat16, g)
    table[0, 2], table[1, 4], table[1, 0] = -1, k.shape[0], 2 ** 31 - 1
    table = torch.cat([table, torch.full((3, room), -3, dtype=torch.int32)], 1)
    q = torch.randn(3 * n, 4, hd, generator=g).bfloat16()
    cache = _cache(k, v, table, lens)
    if op == "attend":
        out, code = S.attend(cache, q.cuda(), 0.09), 52
        ref, _ = R.attend(k, v, table, lens, q, 0.09, 0, 0, page)
    else:
        cu = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32)
        out, code = S.attend_prompt(cache, q.cuda(), cu.cuda(), 0.09), 53
        ref = R.attend_prompt(k, v, table, lens, q, cu, 0.09, 0, 0, page)
    torch.cuda.synchronize()
    assert S.device_error(clear=True) == code and S.device_error() == 0
    _close(out, ref, _tolerance(ref, q, k, v, 0.09, torch.bfloat16))
    table[2, 4] = int(table[2, 3])                             # all pages of sequence 2's list are real now
    cache = _cache(k, v, table[2:, :5].contiguous(), [10 ** 6])
    ref_len = [80]
    cu = torch.tensor([0, n], dtype=torch.int32)
    if op == "attend":
        out = S.attend(cache, q[2:].cuda(), 0.09, window=16)
        ref, _ = R.attend(k, v, table[2:, :5], ref_len, q[2:], 0.09, 16, 0, page)
    else:
        out = S.attend_prompt(cache, q[2 * n:].cuda(), cu.cuda(), 0.09, window=16)
        ref = R.attend_prompt(k, v, table[2:, :5], ref_len, q[2 * n:], cu, 0.09, 16, 0, page)
    torch.cuda.synchronize()
    assert S.device_error(clear=True) == code
    _close(out, ref, _tolerance(ref, q, k, v, 0.09, torch.bfloat16))       # (slots 64 .. 79 lie on page 3 again)


def test_attend_offsets_past_32_bits():
    """A pool of more than 2^32 elements: rows in its last pages are found."""
    from opentars_b200 import serving as S
    n_pages, page, hd = (1 << 32) // (256 * 256) + 40, 256, 256
    k = torch.zeros(n_pages, page, 1, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(11)
    lens = [300]
    table = torch.tensor([[n_pages - 1, n_pages - 30]], dtype=torch.int32)
    for i, p in enumerate(table[0].tolist()):
        k[p] = torch.randn(page, 1, hd, generator=g).bfloat16().cuda()
        v[p] = torch.randn(page, 1, hd, generator=g).bfloat16().cuda()
    cache = S.PagedCache(k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    q = torch.randn(1, 2, hd, generator=g).bfloat16()
    small = torch.tensor([[0, 1]], dtype=torch.int32)
    ks, vs = k[table[0].long().cuda()].cpu(), v[table[0].long().cuda()].cpu()
    ref, _ = R.attend(ks, vs, small, lens, q, 0.06, 0, 0, page)
    tol = _tolerance(ref, q, ks, vs, 0.06, torch.bfloat16)
    _close(S.attend(cache, q.cuda(), 0.06), ref, tol)
    for n in (1, 40):                                          # few rows, and many
        rows = torch.randn(n, 2, hd, generator=g).bfloat16()
        cu = torch.tensor([0, n], dtype=torch.int32)
        want = R.attend_prompt(ks, vs, small, lens, rows, cu, 0.06, 0, 0, page)
        _close(S.attend_prompt(cache, rows.cuda(), cu.cuda(), 0.06), want, _tolerance(want, rows, ks, vs, 0.06, torch.bfloat16))
    S.append(cache, torch.ones(1, 1, hd, device="cuda"), torch.full((1, 1, hd), 2.0, device="cuda"))
    _no_error()
    assert (k[n_pages - 30, 43, 0] == 1).all() and (v[n_pages - 30, 43, 0] == 2).all()


# ------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype,hd,page,kv,seqs", [
    (torch.bfloat16, 128, 16, 2, [(0, 5), (16, 0), (15, 2), (3, 40)]),
    (torch.float16, 64, 32, 3, [(31, 1), (0, 33)]),
    (torch.bfloat16, 256, 256, 1, [(200, 100)])])
def test_append(src, dtype, hd, page, kv, seqs):
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(hd)
    lens = [c + n for c, n in seqs]
    k, v, table = _pools(lens, kv, hd, page, dtype, g)
    cap = table.shape[1] * page
    track = (torch.full((len(lens), kv, cap), 3.0), torch.full((len(lens), kv, cap), -5, dtype=torch.int32),
             torch.tensor([n + 100 for n in lens], dtype=torch.int32))
    cache = _cache(k, v, table, lens, "heads", track)
    cu = [0]
    for _, n in seqs:
        cu.append(cu[-1] + n)
    kn = (torch.randn(cu[-1] + 2, kv, hd, generator=g) * 3).to(src)      # two rows behind the last sequence
    vn = (torch.randn(cu[-1] + 2, kv, hd, generator=g) * 3).to(src)
    S.append(cache, kn.cuda(), vn.cuda(), torch.tensor(cu, dtype=torch.int32).cuda())
    _no_error()
    w, p = track[0].clone(), track[1].clone()
    for b, (c, n) in enumerate(seqs):
        for i in range(n):
            s = c + i
            k[int(table[b, s // page]), s % page] = kn[cu[b] + i].to(dtype)
            v[int(table[b, s // page]), s % page] = vn[cu[b] + i].to(dtype)
            w[b, :, s], p[b, :, s] = 0.0, s + 100
    same = lambda a, b: torch.equal(a.cpu().view(torch.int16), b.view(torch.int16))  # noqa: E731
    assert same(cache.k.contiguous(), k) and same(cache.v.contiguous(), v)
    assert torch.equal(cache.weight.cpu(), w) and torch.equal(cache.pos.cpu(), p)


def test_append_one_row_each_skips_empty_sequences_and_bad_pages():
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(1)
    k, v, table = _pools([17, 0, 16, 5], 1, 64, 16, torch.bfloat16, g)
    table[3, 0] = -7
    cache = _cache(k, v, table, [17, 0, 16, 5])
    rows = torch.randn(4, 2, 64, generator=g).cuda()
    S.append(cache, rows[:, :1], rows[:, 1:])
    torch.cuda.synchronize()
    assert S.device_error(clear=True) == 51
    k[int(table[0, 1]), 0], v[int(table[0, 1]), 0] = rows[0, :1].cpu().bfloat16(), rows[0, 1:].cpu().bfloat16()
    k[int(table[2, 0]), 15], v[int(table[2, 0]), 15] = rows[2, :1].cpu().bfloat16(), rows[2, 1:].cpu().bfloat16()
    assert torch.equal(cache.k.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(cache.v.cpu().view(torch.int16), v.view(torch.int16))


# ------------------------------------------------------------------------------------------- evict
EVICT = [  # head dim, page, kv heads, lengths, budget, sinks, recent, kind of weights
    (128, 16, 2, [33, 32, 5, 0, 100], 32, 4, 8, "plain"),
    (64, 32, 3, [40, 41], 1, 0, 0, "plain"),
    (256, 16, 1, [130], 129, 0, 129, "plain"),
    (128, 64, 2, [3000, 2049], 2048, 4, 500, "ties"),
    (64, 16, 1, [500, 480], 100, 60, 40, "ties"),
    (128, 16, 2, [700, 300], 64, 2, 10, "nonfinite"),
    (64, 16, 1, [70000], 3000, 4, 100, "ties"),
    (64, 256, 2, [5000], 4999, 0, 0, "zeros"),
]


def _weights(kind, shape, g):
    w = torch.exp(2 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.randint(0, 6, shape, generator=g).float() - 1
    if kind == "zeros":
        w = torch.zeros(shape)
        w[..., ::3] = -0.0
    if kind == "nonfinite":
        r = torch.rand(shape, generator=g)
        w = torch.where(r < 0.01, torch.tensor(NAN), w)
        w = torch.where((r > 0.01) & (r < 0.03), torch.tensor(math.inf), w)
        w = torch.where((r > 0.03) & (r < 0.5), torch.tensor(-math.inf), w)
        w = torch.where((r > 0.5) & (r < 0.6), torch.tensor(1e-42), w)
    return w


@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"{c[0]}-{max(c[3])}to{c[4]}-{c[7]}")
@pytest.mark.parametrize("inplace", [True, False], ids=["inplace", "out"])
def test_evict(case, inplace):
    from opentars_b200 import serving as S
    hd, page, kv, lens, budget, sinks, recent, kind = case
    g = torch.Generator().manual_seed(budget)
    k, v, table = _pools(lens, kv, hd, page, torch.bfloat16, g)
    B, cap = len(lens), table.shape[1] * page + 3
    w = _weights(kind, (B, kv, cap), g)
    # a history of evictions: positions are not the slots, and differ between heads
    pos = torch.stack([torch.stack([torch.randperm(cap, generator=g) for _ in range(kv)]) for _ in range(B)]).int()
    seen = torch.full((B,), cap, dtype=torch.int32)
    cache = _cache(k, v, table, lens, "heads", (w, pos, seen))
    lo, wo, po = cache.length, cache.weight, cache.pos
    if not inplace:
        lo, wo, po = torch.full_like(lo, -1), torch.full_like(wo, 5.0), torch.full_like(po, -9)
    want = R.evict(w, pos, lens, seen, budget, sinks, recent)
    S.evict(cache, budget, sinks=sinks, recent=recent, length_out=lo, weight_out=wo, pos_out=po)
    _no_error()
    assert lo.tolist() == [min(n, budget) for n in lens]
    if not inplace:
        assert cache.length.tolist() == lens
    bits = lambda t: t.view(torch.int32)  # noqa: E731
    for b in range(B):
        slot = torch.arange(lens[b])
        pages, rows = table[b].long()[slot // page], slot % page
        for h in range(kv):
            old = torch.tensor(want[b * kv + h], dtype=torch.long)
            n = len(old)
            assert torch.equal(bits(wo[b, h, :n].cpu()), bits(w[b, h, old])), (b, h)
            assert torch.equal(po[b, h, :n].cpu(), pos[b, h, old])
            if not inplace:
                assert (wo[b, h, n:] == 5.0).all() and (po[b, h, n:] == -9).all()
            for pool, was in ((cache.k, k), (cache.v, v)):
                now = pool[pages.cuda(), rows.cuda(), h].cpu().view(torch.int16)
                src = torch.cat([old, torch.arange(n, lens[b])])
                assert torch.equal(now, was[pages[src], rows[src], h].view(torch.int16))


def test_evict_skips_rows_on_bad_pages():
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(3)
    lens, page, hd = [64], 16, 64
    k, v, table = _pools(lens, 1, hd, page, torch.bfloat16, g)
    cap = table.shape[1] * page
    w = torch.arange(cap).float().reshape(1, 1, cap)           # the last slots stay and move to the front
    pos = torch.arange(cap, dtype=torch.int32).reshape(1, 1, cap)
    bad = int(table[0, 2])
    table[0, 2] = -1
    cache = _cache(k, v, table, lens, "heads", (w, pos, torch.tensor(lens, dtype=torch.int32)))
    S.evict(cache, 32)
    torch.cuda.synchronize()
    assert S.device_error(clear=True) == 54
    p = table[0].tolist()
    assert torch.equal(cache.k[p[0]].cpu(), k[p[0]])           # its rows would have come from the bad page
    assert torch.equal(cache.k[p[1]].cpu(), k[p[3]]) and torch.equal(cache.v[p[1]].cpu(), v[p[3]])
    assert torch.equal(cache.k[bad].cpu(), k[bad])
    assert cache.pos[0, 0, :32].tolist() == list(range(32, 64))


# ------------------------------------------------------------------------------------ logits rules
@pytest.mark.parametrize("vocab", [1, 3, 31, 32, 100, 1001, 5000, 70001, 151936])
@pytest.mark.parametrize("inplace", [True, False], ids=["inplace", "out"])
def test_adjust_logits(vocab, inplace):
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(vocab)
    rows, H, NB = 5, 90, 12
    x = torch.randn(rows, vocab, generator=g) * 4
    x[0, vocab // 2] = NAN
    x[1, vocab - 1] = math.inf
    x[2] = -3.4028234663852886e38
    x[3, vocab // 3] = 0.0
    hist = torch.randint(-2, vocab + 2, (rows, H), generator=g, dtype=torch.int32)     # some ids outside
    hist[3, :40] = vocab - 1
    n_hist = torch.tensor([0, H, 50, H, 1], dtype=torch.int32)
    n_prompt = torch.tensor([0, 30, 50, 0, 5], dtype=torch.int32)
    rep, pres, freq = 1 + torch.rand(rows, generator=g), torch.rand(rows, generator=g), torch.rand(rows, generator=g)
    ids = torch.randint(-1, vocab + 1, (rows, NB), generator=g, dtype=torch.int32)
    ids[1] = vocab // 2                                       # one token listed twelve times
    bias = torch.randn(rows, NB, generator=g)
    words = (vocab + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g).int()
    mask[4] = 0                                               # nothing allowed
    tail = vocab % 32
    if tail:
        mask[:, -1] |= -1 << tail                             # bits behind the vocabulary mean nothing
        mask[4, -1] = -1 << tail if tail < 32 else 0
    wide = torch.full((rows, vocab + 3), 1e30)
    wide[:, :vocab] = x
    dev = wide.cuda() if vocab % 2 else x.cuda()
    out = None if inplace else torch.empty(rows, vocab, device="cuda")
    view = dev[:, :vocab]
    c = lambda t: t.cuda()  # noqa: E731
    token = S.adjust_logits(view, history=c(hist), n_history=c(n_hist), n_prompt=c(n_prompt), repetition=c(rep),
                            presence=c(pres), frequency=c(freq), bias_ids=c(ids), bias=c(bias), mask=c(mask), out=out,
                            none=-5)
    _no_error()
    got = (view if inplace else out).cpu()
    t = torch.arange(vocab)
    for r in range(rows):
        allowed = (mask[r][t // 32] >> (t % 32).int()) & 1 == 1
        want, pick = R.adjust(x[r], hist[r], int(n_hist[r]), min(int(n_prompt[r]), int(n_hist[r])), float(rep[r]),
                              float(pres[r]), float(freq[r]), ids[r], bias[r], allowed)
        big = torch.isinf(want.float()) | torch.isnan(want)
        assert torch.equal(torch.isnan(got[r]), torch.isnan(want)) and torch.equal(got[r][big & ~torch.isnan(want)],
                                                                                   want[big & ~torch.isnan(want)].float())
        # five roundings of numbers no larger than |x| rep + freq count + presence + |bias|
        size = x[r].abs().double() * 2 + H + 1 + bias[r].abs().max()
        assert ((got[r].double() - want).abs()[~big] <= 5 * 2.0 ** -24 * size[~big]).all()
        if pick is None:
            assert int(token[r]) == -5
        else:                                                 # the pick of the rounded values, in np.argmax's order
            ok = torch.nonzero(allowed)[:, 0]
            import numpy as np
            assert int(token[r]) == int(ok[int(np.argmax(got[r][ok].numpy()))])
    if not inplace:
        assert torch.equal(torch.nan_to_num(view.cpu()), torch.nan_to_num(x))
    if vocab % 2:
        assert (dev[:, vocab:] == 1e30).all()


def test_adjust_logits_without_rules_is_the_greedy_pick():
    from opentars_b200 import serving as S
    x = torch.randn(3, 4097).cuda()
    was = x.clone()
    assert S.adjust_logits(x).tolist() == was.argmax(1).tolist() and torch.equal(x, was)
    empty = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    assert S.adjust_logits(x, history=empty, repetition=torch.full((3,), 2.0).cuda()).tolist() == was.argmax(1).tolist()
    mask = torch.zeros(129, dtype=torch.int32, device="cuda")  # one mask for all rows
    mask[2] = 1 << 5
    assert S.adjust_logits(x, mask=mask).tolist() == [69] * 3
    hist = torch.tensor([[7, 7, 7]] * 3, dtype=torch.int32, device="cuda")
    y = was.clone()
    S.adjust_logits(y, history=hist, frequency=torch.tensor([0.5, 0.25, 0.0]).cuda())
    assert torch.allclose((was - y)[:, 7].cpu(), torch.tensor([1.5, 0.75, 0.0]), atol=1e-6)
    y[:, 7] = was[:, 7]
    assert torch.equal(y, was)


# --------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_wrappers():
    from opentars_b200 import serving as S
    cache = S.PagedCache.empty(4, 16, 2, 64, 2, 2)
    tracked = S.PagedCache.empty(4, 16, 2, 64, 2, 2, track=True)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    bad = [lambda: S.attend(cache, q.half(), 1.0), lambda: S.attend(cache, q[:1], 1.0), lambda: S.attend(cache, q[:, :3], 1.0),
           lambda: S.attend(cache, q.cpu(), 1.0), lambda: S.attend(cache, q, 1.0, window=-1),
           lambda: S.attend(cache, q, float("nan")), lambda: S.attend(cache, q, 1.0, weight_out=tracked.weight),
           lambda: S.attend(cache, q, 1.0, out=q[:1].expand(2, 4, 64)), lambda: S.attend(cache, q[:, :, ::2], 1.0),
           lambda: S.attend(tracked, q, 1.0, weight_out=tracked.weight[:, :, :8]),
           lambda: S.attend_prompt(cache, q, cu[:2], 1.0), lambda: S.attend_prompt(cache, q, cu.long(), 1.0),
           lambda: S.append(cache, q, q), lambda: S.append(cache, q[:, :2], q[:, :2].float()),
           lambda: S.append(cache, torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")),
           lambda: S.evict(cache, 8), lambda: S.evict(tracked, 0), lambda: S.evict(tracked, 8, sinks=4, recent=5),
           lambda: S.evict(tracked, 8, pos_out=tracked.weight),
           lambda: S.adjust_logits(torch.zeros(2, 10, device="cuda").half()),
           lambda: S.adjust_logits(torch.zeros(1, 10, device="cuda").expand(2, 10)),
           lambda: S.adjust_logits(torch.zeros(2, 10, device="cuda"), repetition=torch.ones(2, device="cuda")),
           lambda: S.adjust_logits(torch.zeros(2, 10, device="cuda"), mask=torch.zeros(2, 2, dtype=torch.int32, device="cuda")),
           lambda: S.adjust_logits(torch.zeros(2, 10, device="cuda"), token=torch.zeros(3, dtype=torch.int32, device="cuda"))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(ValueError):
        S.PagedCache(cache.k, cache.v, cache.table, cache.length, weight=tracked.weight)
    with pytest.raises(ValueError):
        S.PagedCache(cache.k[:, :8], cache.v[:, :8], cache.table, cache.length)


# ----------------------------------------------------------------------------- a run of them together
def _conversation(S, cache, tokens, kv, nh, hd, budget, g, stream=None):
    """Prompt chunks, single tokens and evictions over one cache; returns every output."""
    outs, cu0 = [], torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for n in tokens:
        new = torch.randn(2 * n, kv, hd, generator=g, device="cuda")
        val = torch.randn(2 * n, kv, hd, generator=g, device="cuda")
        q = torch.randn(2 * n, nh, hd, generator=g, device="cuda").bfloat16()
        cache.length.add_(n)
        cache.seen.add_(n)
        S.append(cache, new, val, cu0 * n)
        if n > 1:
            outs.append(S.attend_prompt(cache, q, cu0 * n, hd ** -0.5))
        else:
            outs.append(S.attend(cache, q, hd ** -0.5, weight_out=cache.weight))
        S.evict(cache, budget, sinks=2, recent=16)
    return outs


def test_a_conversation_with_evictions_against_the_definitions():
    """append, attend_prompt, attend with weights and evict in turn, every step's outputs against the
    64-bit forms over the same token history."""
    from opentars_b200 import serving as S
    kv, nh, hd, page, budget = 2, 4, 64, 16, 48
    cache = S.PagedCache.empty(12, page, kv, hd, 2, 6, track=True)
    cache.table.copy_(torch.randperm(12, generator=torch.Generator().manual_seed(0)).reshape(2, 6).int())
    cache.k.fill_(NAN)
    cache.v.fill_(NAN)
    g = torch.Generator(device="cuda").manual_seed(4)
    steps = [30, 1, 1, 25, 1, 1, 1, 40, 1]
    # the model of the cache: per (sequence, head) lists of (key, value, weight, position)
    model = [[[] for _ in range(kv)] for _ in range(2)]
    seen = 0
    for n in steps:
        gs = torch.Generator(device="cuda")
        gs.set_state(g.get_state())
        new = torch.randn(2 * n, kv, hd, generator=gs, device="cuda").bfloat16().cpu()
        val = torch.randn(2 * n, kv, hd, generator=gs, device="cuda").bfloat16().cpu()
        q = torch.randn(2 * n, nh, hd, generator=gs, device="cuda").bfloat16().cpu()
        out = _conversation(S, cache, [n], kv, nh, hd, budget, g)[0].cpu()
        for b in range(2):
            for h in range(kv):
                for i in range(n):
                    model[b][h].append([new[b * n + i, h], val[b * n + i, h], 0.0, seen + i])
        ref = torch.zeros(out.shape, dtype=torch.float64)
        for b in range(2):
            for h in range(kv):
                m = model[b][h]
                kk, vv = torch.stack([e[0] for e in m])[:, None], torch.stack([e[1] for e in m])[:, None]
                for i in range(n):
                    end = len(m) - n + i + 1
                    heads = slice(2 * h, 2 * h + 2)
                    o, p = R.attend_row(q[b * n + i, heads], kk[:end], vv[:end], torch.ones(end, dtype=torch.bool), hd ** -0.5)
                    ref[b * n + i, heads] = o
                    if n == 1:
                        for j in range(end):
                            m[j][2] += float(p[:, j].sum())
        kk = torch.stack([e[0] for e in model[0][0]])[:, None]
        vv = torch.stack([e[1] for e in model[0][0]])[:, None]
        tol = _tolerance(ref, q, torch.cat([kk, new.reshape(-1, 1, hd)]), torch.cat([vv, val.reshape(-1, 1, hd)]), hd ** -0.5,
                         torch.bfloat16)
        _close(out, ref, tol + 2.0 ** -8 * ref.abs().max(), f"step of {n}")
        seen += n
        for b in range(2):
            for h in range(kv):
                m = model[b][h]
                if len(m) > budget:
                    # the device's own sums rank the slots (ties of 64-bit sums may fall otherwise)
                    order = sorted(range(len(m)), key=lambda s: (not (m[s][3] < 2 or m[s][3] >= seen - 16), -m[s][2], s))
                    kept = set(order[:budget])
                    arrive = iter(sorted(s for s in kept if s >= budget))
                    model[b][h] = [m[s] if s in kept else m[next(arrive)] for s in range(budget)]
                assert cache.pos[b, h, :len(model[b][h])].tolist() == [e[3] for e in model[b][h]], (n, b, h)
        assert cache.length.tolist() == [len(model[0][0])] * 2
    _no_error()


def test_captured_calls_replay_and_share_nothing():
    """The calls captured into two CUDA graphs, replayed in turn with eager calls between, on a stream of
    their own: the same bits as eager calls."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(12)
    made = []
    for seed, lens in ((0, [700, 33, 0]), (1, [64, 1500, 129])):
        k, v, table = _pools(lens, 2, 128, 16, torch.bfloat16, g)
        cap = table.shape[1] * 16
        w = torch.rand(3, 2, cap, generator=g)
        pos = torch.arange(cap, dtype=torch.int32).repeat(3, 2, 1)
        cache = _cache(k, v, table, lens, "heads", (w, pos, torch.tensor(lens, dtype=torch.int32)))
        q = torch.randn(3, 4, 128, generator=g).bfloat16().cuda()
        logits = torch.randn(3, 5000, generator=g).cuda()
        hist = torch.randint(0, 5000, (3, 64), generator=g, dtype=torch.int32).cuda()
        cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()
        out = dict(w=torch.zeros_like(cache.weight), w2=torch.zeros_like(cache.weight), p2=torch.zeros_like(cache.pos),
                   n2=torch.zeros_like(cache.length), x=torch.empty_like(logits))
        rep = torch.full((3,), 1.3).cuda()

        def calls(cache=cache, q=q, logits=logits, hist=hist, cu=cu, out=out, rep=rep):
            a = S.attend(cache, q, 0.09, window=600, sinks=4, weight_out=out["w"])
            b = S.attend_prompt(cache, q, cu, 0.09)
            S.evict(cache, 1600, 4, 16, out["n2"], out["w2"], out["p2"])
            t = S.adjust_logits(logits, history=hist, repetition=rep, out=out["x"])
            return [a, b, t, out["w"], out["w2"], out["p2"], out["n2"], out["x"]]
        want = [x.clone() for x in calls()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            got = calls()
        made.append((graph, got, want, calls))
    for _ in range(3):
        for graph, got, want, calls in made:
            for x in got:
                x.zero_()
            graph.replay()
            calls()
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(got, want):
                assert torch.equal(x, y)
    _no_error()


def test_calls_on_two_streams_at_once():
    """Two batches' calls on two streams give what they give one after the other."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(13)
    jobs = []
    for lens in ([3000, 5, 900], [100, 2000, 64]):
        k, v, table = _pools(lens, 2, 64, 16, torch.float16, g)
        cache = _cache(k, v, table, lens)
        q = torch.randn(3, 4, 64, generator=g).half().cuda()
        jobs.append((cache, q, S.attend(cache, q, 0.125).clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(10):
        outs = []
        for (cache, q, _), st in zip(jobs, streams):
            with torch.cuda.stream(st):
                outs.append(S.attend(cache, q, 0.125))
        torch.cuda.synchronize()
        for o, (_, _, want) in zip(outs, jobs):
            assert torch.equal(o, want)
    _no_error()


def test_symbol_addresses_are_reached_through_ctypes():
    """The C entry point itself, as a caller without torch's wrappers uses it."""
    from opentars_b200.serving import Rules_t, lib
    x = torch.randn(2, 300, device="cuda")
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")
    r = Rules_t(logits=x.data_ptr(), out=x.data_ptr(), logits_stride=300, out_stride=300, rows=2, vocab=300,
                token=tok.data_ptr(), none=-1)
    assert lib().tc_adjust_logits(ctypes.byref(r), None) == 0
    torch.cuda.synchronize()
    assert tok.tolist() == x.argmax(1).tolist()


def test_waits_that_run_out_are_recorded():
    """attend_prompt with a poll limit of 0, where every wait for work gives up at once: the call ends, the word
    holds its code, and the next call is right again."""
    from opentars_b200 import serving as S
    from opentars_b200._lib import lib
    g = torch.Generator().manual_seed(14)
    lens = [500, 0, 90]
    k, v, table = _pools(lens, 2, 128, 16, torch.bfloat16, g)
    cache = _cache(k, v, table, lens)
    q = torch.randn(150, 4, 128, generator=g).bfloat16().cuda()
    cu = torch.tensor([0, 80, 80, 150], dtype=torch.int32).cuda()
    call = lambda: S.attend_prompt(cache, q, cu, 0.09)  # noqa: E731
    want = call().clone()
    _no_error()
    was = lib().tc_set_spin_limit(0)
    try:
        call()
        torch.cuda.synchronize()
        assert S.device_error(clear=True) == 55
    finally:
        lib().tc_set_spin_limit(was)
    assert torch.equal(call(), want)
    _no_error()


@pytest.mark.parametrize("name", ["qwen3_small", "gemma3_small"])
def test_the_decode_engine_takes_rules_before_its_picks(name):
    """DecodeEngine.adjust after every step: the changed logits and picks are the rules' on the step's own
    logits, and the following step feeds the changed picks (as a second engine that is given them)."""
    import numpy as np

    from opentars_b200.engine import DecodeEngine
    from tests import fixtures as FX
    from tests.model_runs import build_image
    fx = FX.engine_models()[name]
    rng = np.random.default_rng(3)
    B, V = 3, fx["vocab"]
    prompts = rng.integers(0, V, (B, 4))
    eng, twin = DecodeEngine(build_image(fx), batch=B), DecodeEngine(build_image(fx), batch=B)
    for e in (eng, twin):
        e.reset()
        e.step(prompts, 4)
    hist = torch.zeros(B, 16, dtype=torch.int32, device="cuda")
    hist[:, :4] = torch.from_numpy(prompts).int().cuda()
    n = torch.full((B,), 4, dtype=torch.int32, device="cuda")
    first = n.clone()
    rep, freq = torch.full((B,), 1.7, device="cuda"), torch.full((B,), 0.3, device="cuda")
    for step in range(4):
        plain = twin.logits()
        mask = torch.full((B, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
        top = plain.argmax(1)
        for b in range(B - 1):                                 # the greedy pick of two sequences is forbidden
            mask[b, top[b] // 32] = ~(1 << int(top[b] % 32)) if top[b] % 32 < 31 else 2 ** 31 - 1
        mask[B - 1] = 0                                        # and everything for the third
        eng.adjust(none=7, history=hist, n_history=n, n_prompt=first, repetition=rep, frequency=freq, mask=mask)
        got, picks = eng.logits(), eng.tokens()
        for b in range(B):
            allowed = torch.ones(V, dtype=torch.bool) if b < B - 1 else torch.zeros(V, dtype=torch.bool)
            allowed[top[b]] = False
            want, pick = R.adjust(torch.from_numpy(plain[b]), hist[b].cpu(), int(n[b]), 4, float(rep[b]), 0.0, float(freq[b]),
                                  [], [], allowed)
            assert np.allclose(got[b], want.numpy(), rtol=1e-6, atol=1e-5)
            assert picks[b] == (7 if pick is None else int(np.argmax(got[b])))
        hist[torch.arange(B), n.long()] = torch.from_numpy(picks).cuda()
        n += 1
        eng.step(None)
        twin.step(picks.reshape(B, 1), 1)
        assert np.array_equal(eng.logits().view(np.uint32), twin.logits().view(np.uint32)), step
    with pytest.raises(RuntimeError, match="none"):
        eng.adjust(none=V, mask=mask)
    with pytest.raises(ValueError):
        eng.adjust(repetition=rep)
    with pytest.raises(ValueError):
        eng.adjust(history=hist[:2], repetition=rep)
    eng.close()
    twin.close()


@pytest.mark.parametrize("scale", [-0.11, 0.0])
@pytest.mark.parametrize("n,room", [(2, 700), (130, 0)], ids=["chunk", "tiles"])
def test_negative_and_zero_scales(scale, n, room):
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(15)
    lens, hd, page = [200, n], 64, 16
    k, v, table = _pools(lens, 1, hd, page, torch.float16, g)
    table = torch.cat([table, torch.full((2, room), -1, dtype=torch.int32)], 1)
    q = torch.randn(2 * n, 2, hd, generator=g).half()
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32)
    cache = _cache(k, v, table, lens)
    ref = R.attend_prompt(k, v, table, lens, q, cu, scale, 50, 2, page)
    _close(S.attend_prompt(cache, q.cuda(), cu.cuda(), scale, window=50, sinks=2), ref,
           _tolerance(ref, q, k, v, scale, torch.float16))
    ref, _ = R.attend(k, v, table, lens, q[:2], scale, 50, 2, page)
    _close(S.attend(cache, q[:2].cuda(), scale, window=50, sinks=2), ref, _tolerance(ref, q, k, v, scale, torch.float16))
    _no_error()


@pytest.mark.parametrize("batch", [65, 300, 700])
@pytest.mark.parametrize("n,room", [(0, 0), (1, 900), (3, 900), (40, 0)], ids=["attend", "chunk1", "chunk3", "tiles"])
def test_large_batches(batch, n, room):
    """More sequences than lanes, than threads of a CTA, and several a thread; some are empty."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(batch + n)
    hd, page = 64, 16
    lens = [0 if b % 7 == 3 else max(n, 1) + int(torch.randint(0, 40, (1,), generator=g)) for b in range(batch)]
    lens[batch // 2] = 500
    new = [min(n, x) for x in lens]
    k, v, table = _pools(lens, 1, hd, page, torch.bfloat16, g)
    table = torch.cat([table, torch.full((batch, room), -1, dtype=torch.int32)], 1)
    cache = _cache(k, v, table, lens)
    if n == 0:
        q = torch.randn(batch, 2, hd, generator=g).bfloat16()
        ref, _ = R.attend(k, v, table, lens, q, 0.125, 0, 0, page)
        out = S.attend(cache, q.cuda(), 0.125)
    else:
        cu = torch.tensor([0] + new).cumsum(0).int()
        q = torch.randn(int(cu[-1]), 2, hd, generator=g).bfloat16()
        ref = R.attend_prompt(k, v, table, lens, q, cu, 0.125, 0, 0, page)
        out = S.attend_prompt(cache, q.cuda(), cu.cuda(), 0.125)
    _no_error()
    _close(out, ref, _tolerance(ref, q, k, v, 0.125, torch.bfloat16))


@pytest.mark.parametrize("vocab", [140000, 140001])
@pytest.mark.parametrize("ids", [3000, 20000], ids=["words16", "words32"])
def test_adjust_logits_of_many_rows(vocab, ids):
    """Enough rows for the smaller clusters, a vocabulary of several slices a CTA, and histories on both sides of
    the 16-bit words' limit with tokens counted thousands of times; every value against 64 bits."""
    import numpy as np

    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(ids)
    rows, nb = 20, 2047
    x = torch.randn(rows, vocab, generator=g) * 4
    x[3, 77], x[3, vocab - 3] = NAN, NAN
    x[4] = -math.inf
    hist = torch.randint(0, vocab, (rows, ids), generator=g, dtype=torch.int32)
    hist[:, ::2] = vocab - 1                                   # one token half of the time
    n = torch.randint(ids // 2, ids + 1, (rows,), generator=g, dtype=torch.int32)
    first = (n // 3).int()
    rep, pres, freq = 1 + torch.rand(rows, generator=g), torch.rand(rows, generator=g), torch.rand(rows, generator=g) * 0.01
    bid = torch.randint(0, vocab, (rows, nb), generator=g, dtype=torch.int32)
    bid[:, 1::3] = vocab // 2
    bias = torch.randn(rows, nb, generator=g)
    words = (vocab + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (words,), generator=g).int()
    c = lambda t: t.cuda()  # noqa: E731
    out = torch.empty(rows, vocab, device="cuda")
    token = S.adjust_logits(c(x), history=c(hist), n_history=c(n), n_prompt=c(first), repetition=c(rep), presence=c(pres),
                            frequency=c(freq), bias_ids=c(bid), bias=c(bias), mask=c(mask), out=out, none=-9)
    _no_error()
    got = out.cpu()
    t = torch.arange(vocab)
    allowed = (mask[t // 32] >> (t % 32).int()) & 1 == 1
    for r in range(rows):
        want = x[r].double()
        seen = torch.bincount(hist[r, :int(n[r])].long(), minlength=vocab) > 0
        made = torch.bincount(hist[r, int(first[r]):int(n[r])].long(), minlength=vocab).double()
        want = torch.where(seen, torch.where(want > 0, want / rep[r].double(), want * rep[r].double()), want)
        want = want - freq[r].double() * made - torch.where(made > 0, pres[r].double(), 0.0)
        last = {int(i): float(b) for i, b in zip(bid[r], bias[r])}
        want[list(last)] += torch.tensor(list(last.values()), dtype=torch.float64)
        want[~allowed] = -math.inf
        fin = torch.isfinite(want)
        # five roundings of numbers no larger than these
        size = x[r].abs().double() * 2 + made + 1 + bias[r].abs().max()
        assert torch.equal(torch.isnan(got[r]), torch.isnan(want)) and (got[r][~fin & ~torch.isnan(want)] == -math.inf).all()
        assert ((got[r].double() - want).abs()[fin] <= 5 * 2.0 ** -24 * size[fin]).all(), r
        ok = torch.nonzero(allowed)[:, 0]
        assert int(token[r]) == int(ok[int(np.argmax(got[r][ok].numpy()))]), r


@pytest.mark.parametrize("n", [1, 70], ids=["rows", "tiles"])
def test_heads_first_rows_and_empty_batches(n):
    """q and out in memory as [heads, rows, dim]; a batch of empty sequences; calls of no rows."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(16)
    lens, hd, page = [90, 0, 75], 128, 16
    k, v, table = _pools(lens, 2, hd, page, torch.bfloat16, g)
    cache = _cache(k, v, table, lens)
    new = [n, 0, n]
    cu = torch.tensor([0] + new).cumsum(0).int()
    store = torch.randn(4, 2 * n, hd, generator=g).bfloat16()
    q = store.permute(1, 0, 2)
    ref = R.attend_prompt(k, v, table, lens, q, cu, 0.09, 0, 0, page)
    out = torch.zeros(4, 2 * n, hd, dtype=torch.bfloat16, device="cuda")
    S.attend_prompt(cache, store.cuda().permute(1, 0, 2), cu.cuda(), 0.09, out=out.permute(1, 0, 2))
    _close(out.permute(1, 0, 2), ref, _tolerance(ref, q, k, v, 0.09, torch.bfloat16))
    rows = torch.randn(4, 3, hd, generator=g).bfloat16()
    ref, _ = R.attend(k, v, table, lens, rows.permute(1, 0, 2), 0.09, 0, 0, page)
    one = torch.ones(4, 3, hd, dtype=torch.bfloat16, device="cuda")
    S.attend(cache, rows.cuda().permute(1, 0, 2), 0.09, out=one.permute(1, 0, 2))
    _close(one.permute(1, 0, 2), ref, _tolerance(ref, rows, k, v, 0.09, torch.bfloat16))
    empty = S.PagedCache.empty(2, 16, 2, hd, 3, 2, track=True)
    q0 = torch.randn(3, 4, hd, device="cuda").bfloat16()
    assert (S.attend(empty, q0, 0.09, weight_out=empty.weight) == 0).all() and (empty.weight == 0).all()
    none = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert S.attend_prompt(empty, q0[:0], none, 0.09).shape == (0, 4, hd)
    keep = torch.full_like(q0, 5.0)
    S.attend_prompt(empty, q0, none, 0.09, out=keep)             # no sequence owns a row
    S.append(empty, q0[:, :2], q0[:, :2], none)
    S.append(empty, q0[:, :2], q0[:, :2])                       # lengths of zero: every row is skipped
    S.evict(empty, 4)
    _no_error()
    assert (keep == 5.0).all() and (empty.length == 0).all() and (empty.pos == 0).all()


@pytest.mark.parametrize("vocab,second", [(5000, 2050), (5000, 3000), (151936, 9000), (151936, 140000)])
@pytest.mark.parametrize("how", ["history", "bias"])
def test_adjust_logits_picks_the_first_of_several_nan(vocab, second, how):
    """NaN at two or more tokens, of which the earlier, the later, both or none are listed (a listed token meets a
    thread after the stream of its slice, in any order): the pick is the lowest one, every time."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(vocab + second)
    at = [[5, second], [5, second], [5, second], [5, second], [4, 5, 6, 7, 8, 9, second], [second, 700, 1999, 31, 32]]
    listed = [[5], [second], [5, second], [], [9, 8, 7, 6, second], [second, 1999, 700, 31]]
    x = torch.randn(len(at), vocab, generator=g)
    ids = torch.full((len(at), 40), -1, dtype=torch.int32)
    for r in range(len(at)):
        x[r, at[r]] = NAN
        ids[r, torch.randperm(40, generator=g)[:len(listed[r])]] = torch.tensor(listed[r], dtype=torch.int32)
    rules = dict(history=ids.cuda(), presence=torch.full((len(at),), 0.5).cuda()) if how == "history" else \
        dict(bias_ids=ids.cuda(), bias=torch.ones(len(at), 40).cuda())
    for _ in range(5):
        out = torch.empty_like(x, device="cuda")
        token = S.adjust_logits(x.cuda(), out=out, **rules)
        assert token.tolist() == [min(a) for a in at]
        assert torch.equal(torch.isnan(out.cpu()), torch.isnan(x))
    _no_error()


@pytest.mark.parametrize("dtype,hd,page", [(torch.bfloat16, 128, 64), (torch.bfloat16, 128, 16), (torch.bfloat16, 64, 128),
                                           (torch.bfloat16, 256, 64), (torch.float16, 128, 64), (torch.float16, 256, 16)])
@pytest.mark.parametrize("n,room", [(300, 0), (3, 700)], ids=["tiles", "chunk"])
def test_attend_prompt_rows_whose_scores_are_all_minus_infinity(dtype, hd, page, n, room):
    """Keys with an infinity against queries of one sign: rows that see nothing but scores of -infinity are NaN as
    the formula's 0 / 0 is, rows with a score of +infinity as well, and rows that see one finite score are its."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(21)
    L, far = 400, 390
    k, v, table = _pools([L], 1, hd, page, dtype, g)
    for s in range(far):
        k[int(table[0, s // page]), s % page, 0, 0] = -math.inf
    q = torch.randn(n, 3, hd, generator=g).to(dtype)
    q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
    q[:, 2, 0] = q[:, 2, 0].abs() + 0.5
    table = torch.cat([table, torch.full((1, room), -1, dtype=torch.int32)], 1)
    for length in (far, L):
        cu = torch.tensor([0, n], dtype=torch.int32)
        ref = R.attend_prompt(k, v, table, [length], q, cu, 0.1, 0, 0, page)
        out = S.attend_prompt(_cache(k, v, table, [length]), q.cuda(), cu.cuda(), 0.1)
        _no_error()
        _close(out, ref, _tolerance(ref, q, k, v, 0.1, dtype))
        assert torch.isnan(ref[:, 1]).all() and torch.isnan(ref[:n - (L - far), 0]).all()
    assert n == 3 or torch.isfinite(ref[n - (L - far):, 0]).all()


@pytest.mark.parametrize("op,what", [("prompt", "key"), ("prompt", "value"), ("attend", "key"), ("chunk", "key")])
def test_a_nonfinite_row_that_everyone_sees_costs_no_second_pass(op, what):
    """A NaN in the first key makes every score's sum, and so every output, a NaN; an infinity in the first value makes
    infinities of its column: neither sends the rows to the pass over single keys, which takes hundreds of times as
    long (eight times is the bound, for a busy machine)."""
    from opentars_b200 import serving as S
    B, L, kv, nh, hd, page = (1, 4096, 8, 16, 128, 64) if op == "prompt" else (16, 8192, 8, 16, 128, 16)
    n = dict(prompt=4096, attend=1, chunk=2)[op]
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = B * L // page
    pool = lambda: torch.randn(pages, kv, page, hd, generator=g, device="cuda").bfloat16().permute(0, 2, 1, 3)  # noqa: E731
    cache = S.PagedCache(pool(), pool(), torch.arange(pages, device="cuda").reshape(B, -1).int(),
                         torch.full((B,), L, dtype=torch.int32, device="cuda"))
    q = torch.randn(B * n, nh, hd, generator=g, device="cuda").bfloat16()
    cu = torch.arange(B + 1, device="cuda").int() * n
    call = lambda: S.attend(cache, q, 0.09) if op == "attend" else S.attend_prompt(cache, q, cu, 0.09)  # noqa: E731

    def best():
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times), out
    clean, was = best()
    assert torch.isfinite(was).all()
    first = cache.table[:, 0].long()
    if what == "key":
        cache.k[first, 0] = NAN
    else:
        cache.v[first, 0, :, 3] = math.inf
    slow, out = best()
    _no_error()
    assert slow < 8 * clean, (slow, clean)
    if what == "key":
        assert torch.isnan(out).all()
    else:
        assert (out[:, :, 3] == math.inf).all()
        rest = [i for i in range(hd) if i != 3]
        assert torch.equal(out[:, :, rest], was[:, :, rest])


@pytest.mark.parametrize("op,n", [("attend", 1), ("weights", 1), ("chunk", 2), ("tiles", 8000)])
@pytest.mark.parametrize("hd,page", [(64, 64), (256, 16)])
def test_small_probabilities_of_many_slots_count_in_fp16(op, n, hd, page):
    """One slot draws nearly everything and 60000 others a share below the smallest fp16 number each, together
    more than the output's rounding: they must reach the output as they reach the sum. With values 0 and 1 the
    output is their total share t, rounded to fp16 once: half a step is 2^-11 t. attend_prompt rounds every share to a
    step of 2^-31 of the maximum (2^-24, the probabilities kept 2^7 times as large) once, attend in two parts to
    one of 2^-38: half of that a slot. The exponentials and fp32 sums are allowed 2^-13 t: the exponent, 26, is off
    by 2^-18 at most and each of some 200 additions in a row by 2^-24."""
    from opentars_b200 import serving as S
    L = 60000
    B = 300 if n == 1 else 1                                   # (over the same pages, so that a few warps see a whole one)
    k = torch.zeros(-(-L // page), page, 1, hd, dtype=torch.float16)
    v = torch.ones_like(k)
    k[0, 0, 0, 0], v[0, 0] = 4.5, 0.0
    table = torch.arange(k.shape[0], dtype=torch.int32)[None].expand(B, -1).contiguous()
    q = torch.zeros(B * n, 1, hd, dtype=torch.float16)
    q[:, 0, 0] = 4.0                                           # exp(-18) = 2^-25.97 each
    track = None
    if op == "weights":
        cap = table.shape[1] * page
        track = (torch.zeros(B, 1, cap), torch.zeros(B, 1, cap, dtype=torch.int32), torch.full((B,), L, dtype=torch.int32))
    cache = _cache(k, v, table, [L] * B, "heads", track)
    small = math.exp(-18)
    others = torch.full((B,), L - 1.0).double() if n == 1 else torch.arange(L - n, L).double()
    t = others * small / (1 + others * small)
    if n == 1:
        out = S.attend(cache, q.cuda(), 1.0, weight_out=cache.weight)
    else:
        out = S.attend_prompt(cache, q.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), 1.0)
    _no_error()
    off = (out.double().cpu()[:, 0] - t[:, None]).abs()
    assert (off <= (t * (2.0 ** -11 + 2.0 ** -13) + L * 2.0 ** (-32 if op == "tiles" else -39))[:, None]).all(), off.max()
    if op == "weights":
        w, whole = cache.weight[:, 0].double(), 1 + (L - 1) * small
        assert ((w[:, 0] * whole - 1).abs() < 2.0 ** -13).all()
        assert ((w[:, 1:L] * whole / small - 1).abs() < 2.0 ** -13).all() and (w[:, L:] == 0).all()


def test_whole_numbers_beyond_32_bits_are_refused():
    from opentars_b200 import serving as S
    cache = S.PagedCache.empty(4, 16, 2, 64, 2, 2, track=True)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 10, device="cuda")
    big = 2 ** 32 + 8
    for i, call in enumerate([lambda: S.attend(cache, q, 1.0, window=big), lambda: S.attend(cache, q, 1.0, sinks=big),
                 lambda: S.attend_prompt(cache, q, cu, 1.0, window=big), lambda: S.attend_prompt(cache, q, cu, 1.0, sinks=big),
                 lambda: S.evict(cache, big), lambda: S.evict(cache, big, recent=2 ** 32),
                 lambda: S.adjust_logits(x, none=big), lambda: S.adjust_logits(x, none=-2 ** 31 - 1)]):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_attend_takes_parts_of_one_buffer_that_are_apart():
    """q and out as parts of one buffer: taken where no row of one shares an element with a row of the other, refused
    where one does (in place as well: a row whose output is not finite reads its query again)."""
    import random

    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(31)
    rng = random.Random(31)
    k, v, table = _pools([30, 77, 5], 1, 64, 16, torch.bfloat16, g)
    cache = _cache(k, v, table, [30, 77, 5])
    cu = torch.arange(4).int().cuda()
    plain = torch.randn(3, 2, 64, generator=g).bfloat16().cuda()
    want = [S.attend(cache, plain, 0.1), S.attend_prompt(cache, plain, cu, 0.1)]
    strides = [(128, 64), (64, 192), (256, 128), (384, 64), (128, 512), (256, 64), (72, 320)]
    taken = 0
    for i in range(60):
        row, head = strides[i % len(strides)]
        buf = torch.zeros(4000, dtype=torch.bfloat16, device="cuda")
        part = lambda at: buf.as_strided((3, 2, 64), (row, head, 1), at)  # noqa: E731
        a, b = 8 * rng.randrange(200), 8 * rng.randrange(200)
        if i % 4 == 0:
            b = a + rng.choice([64, 128, -64, 192]) if a >= 64 else a
        of = lambda at: set((at + torch.arange(3)[:, None, None] * row + torch.arange(2)[:, None] * head + torch.arange(64)).flatten().tolist())  # noqa: E731
        q, out = part(a), part(b)
        q.copy_(plain)
        for call, ref in zip((lambda: S.attend(cache, q, 0.1, out=out), lambda: S.attend_prompt(cache, q, cu, 0.1, out=out)), want):
            if of(a) & of(b):
                with pytest.raises(ValueError):
                    call()
            else:
                assert torch.equal(call(), ref)
                taken += 1
    assert 20 < taken < 100
    logits = torch.randn(5, 40, generator=g).cuda()
    with pytest.raises(ValueError):
        S.adjust_logits(logits[:4], out=logits[1:])
    wide = torch.zeros(4, 80, device="cuda")
    wide[:, :40] = logits[:4]
    S.adjust_logits(wide[:, :40], out=wide[:, 40:])
    assert torch.equal(wide[:, 40:], logits[:4]) and torch.equal(wide[:, :40], logits[:4])
    _no_error()


def test_tensors_that_require_a_gradient_are_refused():
    from opentars_b200 import serving as S
    cache = S.PagedCache.empty(4, 16, 2, 64, 2, 2)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 10, device="cuda", requires_grad=True)
    plain = q.detach()
    calls = [lambda: S.attend(cache, q, 1.0), lambda: S.attend_prompt(cache, q, cu, 1.0), lambda: S.append(cache, q[:, :2], q[:, 2:]),
             lambda: S.append(cache, plain[:, :2], q[:, 2:]), lambda: S.adjust_logits(x, out=torch.zeros(2, 10, device="cuda")),
             lambda: S.attend(cache, plain, 1.0, out=torch.zeros_like(q, requires_grad=True))]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="gradient"):
            call()
            pytest.fail(f"call {i} was taken")
    with torch.no_grad():
        for call in calls:
            call()
    _no_error()


@pytest.mark.parametrize("dtype,hd,page", [(torch.bfloat16, 128, 64), (torch.bfloat16, 64, 16), (torch.float16, 256, 64)])
@pytest.mark.parametrize("op,n", [("attend", 1), ("chunk", 3), ("tiles", 300)])
@pytest.mark.parametrize("places", [(0, 3), (6, 7)])
def test_a_score_of_minus_infinity_against_an_infinite_value(op, n, dtype, hd, page, places):
    """Visible slots whose score is -infinity (probability 0) and whose value is infinite: 0 x infinity is NaN in
    their columns, wherever in a block of slots they lie; the other columns are as without them."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(41)
    L = 420
    k, v, table = _pools([L], 1, hd, page, dtype, g)
    slots = [s for s in range(16, 16 + 64) if s % 8 in places]  # visible to every row, in a block that is not masked
    for i, s in enumerate(slots):
        k[int(table[0, s // page]), s % page, 0, 0] = -math.inf
        v[int(table[0, s // page]), s % page, 0, i] = math.inf
    q = torch.randn(n, 2, hd, generator=g).to(dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 0.25
    room = torch.full((1, 700 if op == "chunk" else 0), -1, dtype=torch.int32)
    cache = _cache(k, v, torch.cat([table, room], 1), [L])
    cu = torch.tensor([0, n], dtype=torch.int32)
    ref = R.attend_prompt(k, v, table, [L], q, cu, 0.1, 0, 0, page)
    out = S.attend(cache, q.cuda(), 0.1) if op == "attend" else S.attend_prompt(cache, q.cuda(), cu.cuda(), 0.1)
    _no_error()
    assert torch.isnan(ref[:, :, :len(slots)]).all() and torch.isfinite(ref[:, :, len(slots):]).all()
    _close(out, ref, _tolerance(ref, q, k, v, 0.1, dtype))


@pytest.mark.parametrize("batch", [1, 3])
def test_a_handle_over_the_front_of_the_page_lists(batch):
    """A handle over table[:, :n] of wide page lists does what one over the whole lists does."""
    from opentars_b200 import serving as S
    g = torch.Generator().manual_seed(51)
    lens = [70, 33, 0][:batch]
    k, v, table = _pools([n + 9 for n in lens], 2, 64, 16, torch.float16, g)
    wide = torch.cat([table, torch.full((batch, 500), 10 ** 9, dtype=torch.int32)], 1).cuda()
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    new, q = torch.randn(2 * batch, 2, 64, generator=g).cuda(), torch.randn(2 * batch, 4, 64, generator=g).half().cuda()
    cu = (torch.arange(batch + 1) * 2).int().cuda()
    got = []
    for width in (wide.shape[1], 5):
        w = torch.rand(batch, 2, wide.shape[1] * 16, generator=torch.Generator().manual_seed(1)).cuda()
        pos = torch.arange(wide.shape[1] * 16, dtype=torch.int32).repeat(batch, 2, 1).cuda()
        c = S.PagedCache(_cuda_pool(k, "heads"), _cuda_pool(v, "heads"), wide[:, :width], torch.tensor(lens).int().cuda(), weight=w,
                         pos=pos, seen=torch.tensor(lens).int().cuda())
        c.length.add_(2)
        c.seen.add_(2)
        S.append(c, new, -new, cu)
        a = S.attend_prompt(c, q, cu, 0.125)
        b = S.attend(c, q[:batch], 0.125, weight_out=c.weight)
        S.evict(c, 40, 2, 8)
        got.append([a, b, c.k.contiguous(), c.v.contiguous(), w, pos, c.length])
    _no_error()
    close = _tolerance(got[0][0].double().cpu(), q.cpu(), k, v, 0.125, torch.float16)
    _close(got[1][0], got[0][0].double().cpu(), 2 * close)      # (the room may take the chunk to another kernel)
    for x, y in zip(got[0][1:], got[1][1:]):
        assert torch.equal(x, y)
