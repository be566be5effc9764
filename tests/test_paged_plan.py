"""Host planner of windowed / 8-bit paged attention and the argument checks of its entry
points (no GPU): every query of a plan must attend exactly the tokens the definition names,
once."""
import ctypes as C

import numpy as np
import pytest
import torch

from beam_engine_b200 import _lib
from beam_engine_b200._lib import PagedPlanInfo, lib

ITEM = np.dtype([(n, np.int32) for n in (
    "q_begin", "q_len", "kv_off", "v_begin", "v_end", "n0", "shift", "pos0", "pos_step",
    "sink_end", "window", "flags", "part_base", "p0", "p1", "p2")])


def plan(levels, nq, page, hq, hkv, causal=True, window=-1, sinks=0, sms=148, cap=None):
    L = len(levels)
    arrs = [[np.ascontiguousarray(np.asarray(lv[k], np.int32)) for lv in levels] for k in range(4)]
    ng = np.asarray([len(a) - 1 for a in arrs[0]], np.int32)
    ptrs = [(_lib.P32 * max(L, 1))(*[_lib.ptr32(a) for a in grp]) for grp in arrs]
    info = PagedPlanInfo()
    buf = np.zeros(cap or (1 << 22), np.int32)
    rc = lib().be_paged_plan(L, *ptrs, _lib.ptr32(ng), nq, page, hq, hkv, int(causal), window, sinks,
                             sms, _lib.addr(buf), buf.size, C.byref(info))
    return rc, info, buf


def attended(info, buf, nq, page):
    """Per query: sorted list of (page, slot) that the plan's items show it."""
    items = buf[info.off_work:info.off_work + 16 * info.n_work].view(ITEM)
    kv = buf[info.off_kvlist:info.off_merge_q]
    got = [[] for _ in range(nq)]
    parts = [[] for _ in range(nq)]
    direct = [0] * nq
    for w in items:
        v = np.arange(w["v_begin"], w["v_end"])
        t = np.where(v >= w["n0"], v + w["shift"], v)
        assert w["v_begin"] < w["v_end"] and (t >= 0).all()
        for i in range(w["q_len"]):
            p = int(w["pos0"]) + i * int(w["pos_step"])
            see = np.ones(len(t), bool)
            if w["flags"] & 1:
                see &= t <= p
            if w["window"] >= 0:
                see &= (t >= p - int(w["window"])) | (t < w["sink_end"])
            q = int(w["q_begin"]) + i
            got[q] += [(int(kv[w["kv_off"] + x // page]), int(x % page)) for x in t[see]]
            if w["part_base"] < 0:
                direct[q] += 1
            else:
                parts[q].append(int(w["part_base"]) + i)
    mq = buf[info.off_merge_q:info.off_merge_q + info.n_merge]
    ptr = buf[info.off_merge_ptr:info.off_merge_ptr + info.n_merge + 1]
    mp = buf[info.off_merge_parts:info.total_ints]
    merged = {int(q): sorted(mp[ptr[k]:ptr[k + 1]].tolist()) for k, q in enumerate(mq)}
    for q in range(nq):   # one writer per query: an item, or the merge of its partial rows
        if direct[q]:
            assert direct[q] == 1 and not parts[q] and q not in merged
        else:
            assert merged[q] == sorted(parts[q])
    flat = [p for q in parts for p in q]
    assert len(flat) == len(set(flat)) and (not flat or max(flat) < info.n_parts)
    return [sorted(x) for x in got]


def expected(levels, nq, page, causal, window, sinks):
    seqs = [[] for _ in range(nq)]
    pos, last = [None] * nq, [0] * nq
    for li, (qo, kp, ki, ll) in enumerate(levels):
        for g in range(len(qo) - 1):
            n = kp[g + 1] - kp[g]
            toks = [(ki[kp[g] + j], s) for j in range(n) for s in range(page if j < n - 1 else ll[g])]
            for q in range(qo[g], qo[g + 1]):
                seqs[q] += toks
                if li == len(levels) - 1:
                    pos[q] = len(seqs[q]) - (qo[g + 1] - qo[g]) + q - qo[g]
                    last[q] = len(toks)
    out = []
    for q in range(nq):
        p = pos[q] if pos[q] is not None else len(seqs[q]) - 1
        n = len(seqs[q])
        see = []
        for t in range(n):
            ok = not (causal and t >= n - last[q] and t > p)
            if window >= 0:
                ok = ok and (t >= p - window or t < sinks)
            if ok:
                see.append(tuple(int(x) for x in seqs[q][t]))
        out.append(sorted(see))
    return out


def ragged(rng, n, page, max_q, max_kv, causal_room=True):
    ql = rng.integers(0, max_q + 1, n)
    kl = rng.integers(0, max_kv + 1, n)
    pages = [-(-int(k) // page) for k in kl]
    qo = np.concatenate([[0], np.cumsum(ql)])
    kp = np.concatenate([[0], np.cumsum(pages)])
    ki = rng.permutation(int(kp[-1]) + 3)[:int(kp[-1])]
    ll = [(int(k) - 1) % page + 1 if k else 0 for k in kl]
    return [(qo.tolist(), kp.tolist(), ki.tolist(), ll)], int(qo[-1])


@pytest.mark.parametrize("page", [1, 8, 16, 33])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (8, 8), (12, 4), (16, 1)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (0, 0), (5, 3), (40, 0), (40, 100), (10 ** 9, 4)])
@pytest.mark.parametrize("causal", [True, False])
def test_single_level_plans_attend_the_definition(page, hq, hkv, window, sinks, causal):
    rng = np.random.default_rng(page * 100 + hq + window % 97)
    for trial in range(4):
        # the last trial is long enough to be split
        levels, nq = ragged(rng, 5, page, [1, 3, 40, 2][trial], [20, 60, 90, 3000][trial])
        rc, info, buf = plan(levels, nq, page, hq, hkv, causal, window, sinks)
        assert rc == 0
        assert attended(info, buf, nq, page) == expected(levels, nq, page, causal, window, sinks)


@pytest.mark.parametrize("window,sinks", [(-1, 0), (3, 0), (20, 2), (70, 40), (200, 70)])
def test_cascade_plans_attend_the_definition(window, sinks):
    """Three levels; prefixes of unequal length under one last-level group included."""
    page, rng = 8, np.random.default_rng(window + 2)
    for trial in range(6):
        beams, prompts = 5, 3
        nq = beams * prompts
        pre = rng.integers(1, 6, prompts)
        mid = rng.integers(0, 3, nq // 5 * 2)
        own = rng.integers(0, 3, nq)
        ids = iter(rng.permutation(2000).tolist())

        def level(sizes, groups):
            kp = np.concatenate([[0], np.cumsum(sizes)]).tolist()
            return (groups, kp, [next(ids) for _ in range(kp[-1])],
                    [int(rng.integers(1, page + 1)) if n else 0 for n in sizes])
        split = sorted(rng.choice(np.arange(1, nq), len(mid) - 1, replace=False).tolist())
        levels = [level(pre, list(range(0, nq + 1, beams))), level(mid, [0] + split + [nq]),
                  level(own, list(range(nq + 1)))]
        rc, info, buf = plan(levels, nq, page, 8, 2, True, window, sinks)
        assert rc == 0
        assert attended(info, buf, nq, page) == expected(levels, nq, page, True, window, sinks)


def test_plan_reports_the_size_it_needs():
    levels, nq = ragged(np.random.default_rng(0), 6, 16, 4, 500)
    rc, info, _ = plan(levels, nq, 16, 8, 2, cap=40)
    assert rc == _lib.BE_ECAPACITY and info.total_ints > 40
    rc, info2, buf = plan(levels, nq, 16, 8, 2, cap=info.total_ints)
    assert rc == 0 and info2.total_ints == info.total_ints


@pytest.mark.parametrize("bad", ["sinks", "heads", "last", "indptr", "queries", "group"])
def test_plan_refuses(bad):
    qo, kp, ki, ll = [0, 2], [0, 2], [3, 4], [7]
    hq, hkv, nq, sinks = 8, 2, 2, 0
    if bad == "sinks":
        sinks = -1
    elif bad == "heads":
        hq = 7
    elif bad == "last":
        ll = [17]
    elif bad == "indptr":
        kp = [0, -1]
    elif bad == "queries":
        nq = 1
    elif bad == "group":
        hq, hkv = 129 * 2, 2
    rc, _, _ = plan([(qo, kp, ki, ll)], nq, 16, hq, hkv, sinks=sinks)
    assert rc == _lib.BE_EINVAL


@pytest.mark.parametrize("qo,kp", [([0, 5000, 2], [0, 1, 2]), ([0, 3, 2], [0, 1, 2]), ([0, -3, 2], [0, 1, 2]),
                                   ([0, 1, 2], [0, 400, 2]), ([0, 2, 5000], [0, 1, 2]),
                                   ([0, 1, 2], [0, 2, 1])])
def test_indptrs_that_do_not_ascend(qo, kp):
    """Refused before anything is indexed by them (a later end may be back in range)."""
    assert plan([(qo, kp, [3, 4], [5, 5])], 2, 16, 8, 2)[0] == _lib.BE_EINVAL
    two = [([0, 1, 2], [0, 1, 2], [3, 4], [5, 5]), (qo, kp, [3, 4], [5, 5])]
    assert plan(two, 2, 16, 8, 2)[0] == _lib.BE_EINVAL


def test_empty_plan():
    rc, info, buf = plan([([0], [0], [], [])], 0, 16, 8, 2)
    assert rc == 0 and info.n_work == 0 and info.n_merge == 0


def _append(**kw):
    a = dict(k=16, v=16, ks=1, vs=1, b=16, pos=16, rp=None, ki=16, kp=16, n=4, f=None, cache=16,
             scale=16, pages=8, ps=16, h=2, d=64, dt=_lib.BE_BF16, cdt=_lib.BE_E4M3, ws=None, wn=0)
    a.update(kw)
    order = "k v ks vs b pos rp ki kp f cache scale ws wn stream n pages ps h d dt cdt".split()
    a["stream"] = 0
    return lib().be_rope_append_paged_kv(
        _lib.ROPE_APPEND_ARGS.pack(*[a[x] or 0 for x in order], 0))


@pytest.mark.parametrize("kw,rc", [
    (dict(d=80), _lib.BE_EINVAL), (dict(ps=257), _lib.BE_EINVAL), (dict(h=65), _lib.BE_EINVAL),
    (dict(scale=None), _lib.BE_EINVAL), (dict(cdt=_lib.BE_F16), _lib.BE_EINVAL),
    (dict(cdt=_lib.BE_BF16), _lib.BE_EINVAL), (dict(k=None), _lib.BE_EINVAL),
    (dict(b=None), _lib.BE_EINVAL), (dict(n=-1), _lib.BE_EINVAL), (dict(dt=_lib.BE_E4M3), _lib.BE_EINVAL),
    (dict(cache=20), _lib.BE_EINVAL), (dict(n=513), _lib.BE_ECAPACITY),
    (dict(n=513, ws=16, wn=100), _lib.BE_ECAPACITY), (dict(n=513, ws=20, wn=4096), _lib.BE_EINVAL),
    (dict(n=0), _lib.BE_OK)])
def test_append_arguments(kw, rc):
    assert _append(**kw) == rc


@pytest.mark.parametrize("kw", [
    dict(dt=_lib.BE_F32), dict(cdt=_lib.BE_F16), dict(d=80), dict(scale=None), dict(hq=258),
    dict(q=None), dict(q=8), dict(parts=1), dict(qs=4), dict(narrow=-1), dict(rows=17),
    dict(pages=1 << 26), dict(pages=2 ** 31 - 1)])
def test_run_refuses(kw):
    a = dict(q=16, qs=512, cache=16, scale=16, hq=4, d=64, dt=_lib.BE_BF16, cdt=_lib.BE_E4M3,
             parts=0, narrow=1, rows=4, pages=8)
    a.update(kw)
    rc = lib().be_paged_attn_run(_lib.PAGED_ATTN_ARGS.pack(
        16, a["q"] or 0, a["qs"], a["cache"], a["scale"] or 0, 16, 512, 0, 0, 0, 0, 0, a["narrow"],
        a["rows"], 0, a["parts"], 16, a["pages"], a["hq"], 2, a["d"], a["dt"], a["cdt"], 1.0, 0))
    assert rc == _lib.BE_EINVAL


def test_host_tensors_are_refused():
    from beam_engine_b200.page import append_paged_kv_cache, read_paged_kv_cache
    pool = torch.zeros((2, 2, 16, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.zeros((2, 2, 2))
    rows, one = torch.zeros((1, 2, 64)), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_paged_kv_cache(rows, rows, one, one, pool, one, one, kv_scale=scale)
    with pytest.raises(RuntimeError, match="CUDA"):
        read_paged_kv_cache(pool, one, scale)
    with pytest.raises(ValueError, match="float8"):
        read_paged_kv_cache(torch.zeros((2, 2, 16, 2, 64)), one, scale)


def test_argument_blocks_match_the_header():
    """The packed blocks have the sizes that the C structs of the header have, and no block is refused."""
    import os
    import re
    src = open(os.path.join(os.path.dirname(__file__), "..", "include", "beam_b200.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    for name, packed in (("be_rope_append_args", _lib.ROPE_APPEND_ARGS),
                         ("be_paged_attn_args", _lib.PAGED_ATTN_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
        fmt = ""
        for decl in body.split(";"):
            fields = decl.strip()
            if fields:
                kind = "Q" if "*" in fields else "q" if "int64_t" in fields else "f" if "float" in fields else "i"
                fmt += kind * len(fields.split(","))
        assert packed.size == sum({"Q": 8, "q": 8, "i": 4, "f": 4}[c] for c in fmt)
        plain = re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), packed.format[1:])
        assert plain == fmt
    assert lib().be_paged_attn_run(None) == _lib.BE_EINVAL
    assert lib().be_rope_append_paged_kv(None) == _lib.BE_EINVAL


@pytest.mark.parametrize("qo,kp,ki,last,ok", [
    ([0, 1, 2], [0, 2, 3], [4, 5, 6], [1, 1], True), ([0], [0], [], [], True), ([0], [], [], [], True),
    ([0, 1, 2], [0, 2, 3], [4, 5, 6, 7], [1, 1, 1], True), ([], [], [], [], False),
    ([0, 1, 2], [0, 2], [4, 5, 6], [1, 1], False), ([0, 1, 2], [0, 2, 3], [4, 5], [1, 1], False),
    ([0, 1, 2], [0, 2, 3], [4, 5, 6], [1], False), ([0, 1], [], [], [], False)])
def test_arrays_shorter_than_the_indptrs_say_are_refused(qo, kp, ki, last, ok):
    from beam_engine_b200.cascade import check_level_sizes
    good = ([0, 1], [0, 1], [3], [2])
    for levels in ([(qo, kp, ki, last)], [good, (qo, kp, ki, last)]):
        arrs = [[np.asarray(lv[k], np.int32) for lv in levels] for k in range(4)]
        if ok:
            check_level_sizes(arrs)
        else:
            with pytest.raises(ValueError, match="level"):
                check_level_sizes(arrs)


NO_MEMORY = """
import resource, sys
import numpy as np
sys.path[:0] = {path}
from test_paged_plan import plan
vm = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (vm + (256 << 20), vm + (256 << 20)))
n = 1 << 27                                       # lists of 2^27 queries: 1 GB each
sys.exit(plan([([0, 0], [0, 1], [0], [1])], n, 16, 8, 2, cap=64)[0])
"""


def test_no_memory_is_a_status():
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    p = subprocess.run([sys.executable, "-c", NO_MEMORY.format(path=[here, os.path.dirname(here)])],
                       capture_output=True, text=True, timeout=300)
    assert p.returncode == _lib.BE_ENOMEM, p.stderr
