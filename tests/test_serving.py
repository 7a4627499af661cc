"""The serving operators' host side on the CPU: exported symbols, the C structures' layout, every
refusal before any device call, and workspace sizes. No device is needed: pointers are never
dereferenced by the checks."""
import ctypes
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def L():
    from opentars_b200 import build
    build.build()
    from opentars_b200.serving import lib
    return lib()


def test_library_exports_every_serving_symbol(L):
    header = (ROOT / "include" / "tarscuda_serve.h").read_text()
    from opentars_b200.serving import SERVE_SIGNATURES
    declared = set(re.findall(r"^(?:int|uint64_t) (tc_[a-z_0-9]+)\s*\(", header, re.M))
    assert declared == set(SERVE_SIGNATURES), declared ^ set(SERVE_SIGNATURES)
    for name in declared:
        assert hasattr(L, name), name


def test_structures_match_the_header():
    """Field names and order of the ctypes structures against the header's."""
    from opentars_b200 import serving as S
    header = (ROOT / "include" / "tarscuda_serve.h").read_text()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    kinds = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32}
    for name, cls in (("tc_kv_cache", S.Cache_t), ("tc_logits_rules", S.Rules_t)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", header).group(1)
        fields = []
        for line in body.split(";"):
            line = line.strip()
            if not line:
                continue
            m = re.match(r"(?:const )?(\w+)\s*(.*)", line)
            for part in m.group(2).split(","):
                star = "*" in line
                fields.append((part.replace("*", "").strip(), ctypes.c_void_p if star else kinds[m.group(1)]))
        assert fields == [tuple(f) for f in cls._fields_]


def _cache(**kw):
    from opentars_b200.serving import Cache_t
    a = 1 << 20
    d = dict(k=a, v=a, page_stride=16 * 128, slot_stride=128, head_stride=16 * 128, n_pages=8, page_size=16, n_kv=1,
             head_dim=128, dtype=1, batch=2, max_pages=4, table=a, table_stride=4, length=a, weight=None, pos=None,
             track_stride=0, seen=None)
    d.update(kw)
    return Cache_t(**d)


TRACK = dict(weight=1 << 20, pos=1 << 20, seen=1 << 20, track_stride=64)
BAD_CACHES = [dict(k=None), dict(v=None), dict(table=None), dict(length=None), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2),
              dict(page_stride=2049), dict(slot_stride=-128), dict(head_stride=4), dict(n_pages=0), dict(page_size=8),
              dict(page_size=24), dict(page_size=512), dict(n_kv=0), dict(head_dim=96), dict(head_dim=512), dict(dtype=0),
              dict(dtype=2), dict(batch=0), dict(max_pages=0), dict(max_pages=1 << 28), dict(table_stride=3),
              dict(weight=1 << 20), dict(TRACK, seen=None), dict(TRACK, track_stride=63)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: ",".join(d))
def test_bad_caches_are_refused(L, bad):
    c = ctypes.byref(_cache(**bad))
    p = 1 << 20
    assert L.tc_kv_append(c, p, p, 1, 128, 128, None, 1, None) == -2
    assert L.tc_attend(c, p, 256, 128, p, 256, 128, 2, 1.0, 0, 0, None, None, 0, None) == -2
    assert L.tc_attend_prompt(c, p, 256, 128, p, 256, 128, 2, p, 1, 1.0, 0, 0, p, 1 << 30, None) == -2
    assert L.tc_kv_evict(c, 16, 0, 0, p, p, p, p, 1 << 30, None) == -2
    assert L.tc_attend_workspace(c, 2, 1) == 0 and L.tc_kv_evict_workspace(c, 16) == 0
    assert L.tc_attend_prompt_workspace(c, 2, 1, 0, 0) == 0


def test_bad_calls_are_refused(L):
    p = 1 << 20
    c = ctypes.byref(_cache(**TRACK))
    two = ctypes.byref(_cache(n_kv=2, **TRACK))
    assert L.tc_kv_append(None, p, p, 1, 128, 128, None, 1, None) == -2
    append = [(None, p, 1, 128, 128, p, 1), (p, None, 1, 128, 128, p, 1), (p, p, 2, 128, 128, p, 1),
              (p, p, 1, 132, 128, p, 1), (p, p, 0, 128, -4, p, 1), (p + 8, p, 0, 128, 128, p, 1), (p, p, 1, 128, 128, p, -1),
              (p, p, 1, 128, 128, None, 3)]
    for a in append:
        assert L.tc_kv_append(c, *a, None) == -2, a
    assert L.tc_kv_append(c, None, None, 1, 0, 0, None, 0, None) == 0          # nothing to do
    ws = L.tc_attend_workspace(c, 2, 1)
    assert ws > 0
    ok = dict(q=p, qr=256, qh=128, out=p, orow=256, oh=128, nh=2, scale=1.0, window=0, sinks=0, w=p, ws=p, n=ws)
    for bad in (dict(q=None), dict(out=None), dict(q=p + 8), dict(out=p + 4), dict(qr=4), dict(qh=-128), dict(orow=2),
                dict(oh=4), dict(nh=0), dict(nh=1 << 20), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(window=-1), dict(sinks=-1), dict(ws=None), dict(ws=p + 16), dict(n=ws - 1)):
        a = dict(ok, **bad)
        assert L.tc_attend(c, *(a[k] for k in ok), None) == -2, bad
    assert L.tc_attend(two, *(dict(ok, nh=3)[k] for k in ok), None) == -2       # heads not a multiple
    assert L.tc_attend(ctypes.byref(_cache()), *(ok[k] for k in ok), None) == -2  # weights of a cache without them
    prompt = [(None, p, 1), (p, None, 1), (p, p, -1), (p, p, (1 << 28) + 1)]
    for q, cu, n in prompt:
        assert L.tc_attend_prompt(c, q, 256, 128, p, 256, 128, 2, cu, n, 1.0, 0, 0, p, 1 << 30, None) == -2, (q, cu, n)
    assert L.tc_attend_prompt(c, None, 0, 0, None, 0, 0, 2, p, 0, 1.0, 0, 0, None, 0, None) == 0
    long = ctypes.byref(_cache(n_pages=1000, max_pages=1000, table_stride=1000))
    n = L.tc_attend_prompt_workspace(long, 2, 3, 0, 0)
    assert n > 0 and L.tc_attend_prompt_workspace(long, 2, 5000, 0, 0) == 0    # few rows, many rows
    assert L.tc_attend_prompt_workspace(long, 2, 3, -1, 0) == 0 and L.tc_attend_prompt_workspace(long, 2, 3, 0, -1) == 0
    for ws, size in ((None, n), (p + 16, n), (p, n - 1)):
        assert L.tc_attend_prompt(long, p, 256, 128, p, 256, 128, 2, p, 3, 1.0, 0, 0, ws, size, None) == -2
    n = L.tc_kv_evict_workspace(c, 16)
    assert n > 0
    evict = [(0, 0, 0, p, p, p, p, n), (16, -1, 0, p, p, p, p, n), (16, 0, -1, p, p, p, p, n), (16, 9, 8, p, p, p, p, n),
             (16, 0, 0, None, p, p, p, n), (16, 0, 0, p, None, p, p, n), (16, 0, 0, p, p, None, p, n),
             (16, 0, 0, p, p, p, None, n), (16, 0, 0, p, p, p, p + 8, n), (16, 0, 0, p, p, p, p, n - 1),
             (16, 2 ** 31 - 1, 2 ** 31 - 1, p, p, p, p, n)]
    for a in evict:
        assert L.tc_kv_evict(c, *a, None) == -2, a
    assert L.tc_kv_evict(ctypes.byref(_cache()), 16, 0, 0, p, p, p, p, n, None) == -2


def test_bad_rules_are_refused(L):
    from opentars_b200.serving import Rules_t
    p = 1 << 20
    ok = dict(logits=p, out=p, logits_stride=100, out_stride=100, rows=2, vocab=100, history=p, history_stride=8,
              max_history=8, bias_ids=p, bias=p, bias_stride=4, n_bias=4, mask=p, mask_stride=4, token=p)
    for bad in (dict(logits=None), dict(out=None), dict(logits_stride=99), dict(out_stride=99), dict(rows=0), dict(vocab=0),
                dict(rows=(1 << 24) + 1), dict(vocab=(1 << 28) + 1), dict(max_history=1 << 20, history_stride=1 << 21),
                dict(history_stride=7), dict(max_history=-1), dict(bias=None), dict(bias_ids=None), dict(n_bias=2048,
                bias_stride=4096), dict(bias_stride=3), dict(n_bias=-1), dict(mask_stride=3), dict(mask_stride=-1),
                dict(history=None, repetition=p), dict(history=None, presence=p), dict(history=None, frequency=p),
                dict(history=None, n_history=p), dict(history=None, n_prompt=p)):
        assert L.tc_adjust_logits(ctypes.byref(Rules_t(**dict(ok, **bad))), None) == -2, bad
    assert L.tc_adjust_logits(None, None) == -2


def test_the_wrappers_refuse_tensors_they_cannot_take():
    """ValueError before any library call (CPU tensors: no device is touched)."""
    import torch

    from opentars_b200 import serving as S
    pool = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        S.PagedCache(pool, pool, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="bf16 or fp16"):
        S.PagedCache(pool.float(), pool.float(), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="two pools"):
        S.PagedCache(pool, pool[:2], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="logits"):
        S.rules_of(torch.zeros(1, 10))
    t = torch.zeros(3, 4, 64)
    assert S._apart(t) and S._apart(t.permute(1, 0, 2)) and S._apart(t[:, :1]) and S._apart(t[:1])
    assert not S._apart(t[:1].expand(3, 4, 64)) and not S._apart(torch.zeros(300)[:].as_strided((2, 2, 64), (64, 64, 1)))


def test_pools_whose_rows_share_memory_are_refused(L):
    """A stride of 0 over several entries (a pool expanded over its heads), and strides that step into the next
    row: refused by every call and by the handle; any nesting of the dimensions is taken."""
    import torch

    from opentars_b200 import serving as S
    p = 1 << 20
    ok = dict(n_kv=2, n_pages=8, page_size=64, page_stride=2 * 64 * 128, head_stride=64 * 128, slot_stride=128)
    for bad in (dict(head_stride=0), dict(slot_stride=0), dict(page_stride=0), dict(slot_stride=64), dict(head_stride=128),
                dict(page_stride=64 * 128), dict(head_stride=63 * 128), dict(slot_stride=256), dict(page_stride=128),
                dict(n_pages=2 ** 31 - 1, page_stride=1 << 39, head_stride=(1 << 39) + 128)):
        c = ctypes.byref(_cache(**dict(ok, **bad), **TRACK, max_pages=1, table_stride=1))
        assert L.tc_kv_append(c, p, p, 1, 256, 128, None, 1, None) == -2, bad
        assert L.tc_attend(c, p, 256, 128, p, 256, 128, 2, 1.0, 0, 0, None, p, 1 << 30, None) == -2, bad
        assert L.tc_attend_prompt(c, p, 256, 128, p, 256, 128, 2, p, 1, 1.0, 0, 0, p, 1 << 30, None) == -2, bad
        assert L.tc_kv_evict(c, 16, 0, 0, p, p, p, p, 1 << 30, None) == -2, bad
        assert L.tc_attend_workspace(c, 2, 0) == 0, bad
    for good in (dict(), dict(slot_stride=256, head_stride=128), dict(slot_stride=256, head_stride=64 * 256, page_stride=2 * 64 * 256),
                 dict(page_stride=128, slot_stride=8 * 128, head_stride=8 * 64 * 128), dict(n_kv=1, head_stride=0),
                 dict(n_pages=1, page_stride=0), dict(page_stride=(64 * 2 - 1) * 128 + 136)):
        c = ctypes.byref(_cache(**dict(ok, **good), max_pages=1, table_stride=1))
        assert L.tc_attend_workspace(c, 2, 0) > 0, good
    pool = torch.zeros(4, 64, 2, 128, dtype=torch.bfloat16)
    table, length = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for bad in (pool[:, :, :1].expand(4, 64, 2, 128), pool[:1].expand(4, 64, 2, 128), pool[:, :1].expand(4, 64, 2, 128),
                pool.as_strided((4, 64, 2, 128), (16384, 256, 64, 1))):
        with pytest.raises(ValueError, match="apart"):
            S.PagedCache(bad, bad, table, length)
    for good in (pool, pool.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), pool[:, :, :1], pool[:1]):
        with pytest.raises(ValueError, match="CUDA"):           # everything else about it is right
            S.PagedCache(good, good, table, length)


def test_whole_numbers_that_32_bits_do_not_hold_are_refused():
    """ctypes drops the higher bits without a word: a budget of 2^32 + 8 would cut a cache to 8 slots."""
    import torch

    from opentars_b200 import serving as S
    S._whole(0, window=0, sinks=2 ** 31 - 1)
    S._whole(-2 ** 31, none=-2 ** 31)
    for low, v in ((0, 2 ** 31), (0, 2 ** 32 + 8), (0, -1), (1, 0), (-2 ** 31, -2 ** 31 - 1), (0, 2 ** 64)):
        with pytest.raises(ValueError, match="window"):
            S._whole(low, window=v)
    for none in (2 ** 31, 2 ** 32 + 7, -2 ** 31 - 1):
        with pytest.raises(ValueError, match="none"):
            S.rules_of(None, shape=(2, 10), device=torch.device("cpu"), none=none)
    assert S.rules_of(None, shape=(2, 10), device=torch.device("cpu"), none=-5).none == -5


def test_outputs_that_share_memory_with_inputs_are_refused(L):
    from opentars_b200.serving import Rules_t
    p = 1 << 20
    c = ctypes.byref(_cache(**TRACK))                          # 2 sequences, a head of 128, 64 slots tracked
    # (q's strides, out's start in elements and strides)
    for qr, qh, at, orow, oh in ((256, 128, 0, 256, 128), (256, 128, 128, 256, 128), (256, 128, -384, 256, 128), (256, 128, 504, 256, 128),
                                 (512, 128, 512, 512, 128), (512, 128, 128, 512, 128), (128, 512, 384, 128, 512),
                                 (512, 256, 120, 512, 256), (512, 128, 256, 256, 128), (0, 128, 128, 256, 128)):
        out = p + 2 * at
        assert L.tc_attend(c, p, qr, qh, out, orow, oh, 2, 1.0, 0, 0, None, p, 1 << 30, None) == -2, (qr, qh, at)
        assert L.tc_attend_prompt(c, p, qr, qh, out, orow, oh, 2, p, 2, 1.0, 0, 0, p, 1 << 30, None) == -2, (qr, qh, at)
    n = 2 * 64
    for at in (4, -4, 4 * (n - 1), -4 * (n - 1)):
        assert L.tc_attend(c, p, 256, 128, p + 4096, 256, 128, 2, 1.0, 0, 0, p + at, p, 1 << 30, None) == -2, at
        assert L.tc_kv_evict(c, 16, 0, 0, p, p + at, p, p, 1 << 30, None) == -2, at
        assert L.tc_kv_evict(c, 16, 0, 0, p, p, p + at, p, 1 << 30, None) == -2, at
    assert L.tc_kv_evict(c, 16, 0, 0, p + 4, p, p, p, 1 << 30, None) == -2
    for at, stride, ostride in ((4, 100, 100), (-4, 100, 100), (400, 100, 100), (0, 100, 104), (200, 200, 200), (400, 200, 208)):
        r = Rules_t(logits=p, out=p + at, logits_stride=stride, out_stride=ostride, rows=2, vocab=100)
        assert L.tc_adjust_logits(ctypes.byref(r), None) == -2, (at, stride)


def test_the_engines_rules_take_no_outputs():
    """DecodeEngine.adjust works on the engine's own logits and picks: out and token, which it would never
    write, are not among its keywords (no engine is needed to refuse them)."""
    import inspect

    from opentars_b200 import serving as S
    from opentars_b200.engine import DecodeEngine
    for name in ("out", "token", "logits", "no_such_rule"):
        with pytest.raises(TypeError, match=name):
            DecodeEngine.adjust(object(), **{name: None})
    rules = set(inspect.signature(S.rules_of).parameters) - {"logits", "out", "token", "shape", "device"}
    assert set(inspect.signature(DecodeEngine.adjust).parameters) == rules | {"self"}


def test_tensors_that_require_a_gradient_are_refused():
    from types import SimpleNamespace

    import torch

    from opentars_b200 import serving as S
    cpu = torch.device("cpu")
    cache = SimpleNamespace(head_dim=64, n_kv=2, device=cpu, dtype=torch.bfloat16)
    plain = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, requires_grad=True)
    S._attend_args(cache, plain, None, 0, 0)
    S._attend_args(cache, q.detach(), None, 0, 0)
    for args in ((q, None), (plain, q), (2 * q, None)):
        with pytest.raises(ValueError, match="gradient"):
            S._attend_args(cache, *args, 0, 0)
    for k, v in ((q, plain), (plain, q)):
        with pytest.raises(ValueError, match="gradient"):
            S.append(cache, k[:, :2], v[:, 2:], torch.zeros(2))
    with torch.no_grad():
        S._attend_args(cache, q, None, 0, 0)
