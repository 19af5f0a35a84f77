"""Caches in fewer bits without a GPU: what the entry points refuse, what they
do nothing for, sizes, and the kernels that calls take, over a pretended HIP
runtime (tests/fake_kvq.cpp). Everything here runs on the CPU."""
import os
import re
import shutil
import subprocess

import pytest

import orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
INVALID, UNSUPPORTED, NOINIT = -1, -2, -4
F16, Q8, Q4 = orc.F16, orc.KV_Q8, orc.KV_Q4


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime_api.h")):
        pytest.skip("no compiler or no HIP headers")
    exe = str(tmp_path_factory.mktemp("fake") / "fake_kvq")
    lib = os.path.dirname(orc.HIP_LIB)
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-rdynamic", "-I", os.path.join(ROCM, "include"),
                    os.path.join(ROOT, "tests", "fake_kvq.cpp"), "-o", exe, "-L", lib, "-lorc_hip",
                    f"-Wl,-rpath,{lib}", "-Wl,--allow-shlib-undefined", "-ldl", "-lpthread"], check=True)

    def run(*lines, init=True):
        """(status, kernels, message) of each call"""
        text = "\n".join((["init"] if init else []) + [" ".join(map(str, x)) for x in lines]) + "\n"
        r = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, (r.returncode, r.stderr)
        out = []
        for line in r.stdout.splitlines()[init:]:
            head, _, msg = line.partition(" | ")
            out.append((int(head.split()[0]), head.split()[1:], msg))
        assert len(out) == len(lines)
        return out

    return run


def test_nothing_before_init(call):
    calls = [["table", 1, 0, 8, 64, 1e4, "-"], store(), load(), attn()]
    assert [c[0] for c in call(*calls, init=False)] == [NOINIT] * 4


def table(p=1, pos0=0, n=100, rot=64, base=1e4, sc="-"):
    return ["table", p, pos0, n, rot, base, sc]


@pytest.mark.parametrize("args", [
    {"p": 0}, {"p": 1, "pos0": -1}, {"n": -1}, {"rot": 0}, {"rot": 63}, {"rot": 130}, {"base": 1.0}, {"base": -3},
    {"pos0": 2 ** 31 - 5, "n": 6}, {"sc": "4 2 1 4 100 0"}, {"sc": "-1 2 1 4 100 0"}, {"sc": "1 0.5 0 0 0 0"},
    {"sc": "2 2 0 4 100 0"}, {"sc": "2 2 4 4 100 0"}, {"sc": "2 2 1 4 0 0"}, {"sc": "3 2 1 4 100 -1"}])
def test_table_refuses(call, args):
    rc, kernels, msg = call(table(**args))[0]
    assert rc == INVALID and not kernels and msg.startswith("rope_table")


def test_table_calls(call):
    a, b, c = call(table(), table(n=0, p=0), table(sc="3 4 1 32 32768 0"))
    assert a[0] == 0 and len(a[1]) == 1 and b == (0, [], "") and c[0] == 0 and len(c[1]) == 1


def store(type=Q8, qkv=1, ld=None, ns=2, nt=3, h=4, kv=2, hd=64, lay=0, rot=64, rope=1, ro=0, pos=1, off=0, q=1, ldq=None,
          k=1, v=1, ctx=128):
    return ["store", type, qkv, (h + 2 * kv) * hd if ld is None else ld, ns, nt, h, kv, hd, lay, rot, rope, ro, pos, off, q,
            h * hd if ldq is None else ldq, k, v, ctx]


@pytest.mark.parametrize("args,code", [
    ({"type": 8}, UNSUPPORTED), ({"type": 0}, UNSUPPORTED), ({"hd": 96}, UNSUPPORTED), ({"hd": 256}, UNSUPPORTED),
    ({"qkv": 0}, INVALID), ({"q": 0}, INVALID), ({"k": 0}, INVALID), ({"v": 0}, INVALID), ({"rope": 0}, INVALID),
    ({"qkv": 2}, INVALID), ({"q": 2}, INVALID), ({"k": 2}, INVALID), ({"v": 2}, INVALID), ({"rope": 2}, INVALID),
    ({"ld": 508}, INVALID), ({"ld": 514}, INVALID), ({"ldq": 252}, INVALID), ({"ldq": 258}, INVALID), ({"ns": -1}, INVALID),
    ({"nt": -1}, INVALID), ({"h": 0}, INVALID), ({"kv": 0}, INVALID), ({"lay": 2}, INVALID), ({"rot": 63}, INVALID),
    ({"rot": 66}, INVALID), ({"rot": -2}, INVALID), ({"ro": -1}, INVALID), ({"ctx": 0}, INVALID), ({"ctx": 100}, INVALID),
    ({"pos": 0, "off": 126}, INVALID), ({"pos": 0, "off": -1}, INVALID), ({"q": 3}, INVALID),
    ({"ns": 1 << 15, "nt": 1 << 15, "ctx": 1 << 15}, INVALID), ({"ns": 1 << 30, "nt": 1 << 30, "ctx": 1 << 30}, INVALID),
    ({"ns": 0x7fffffff, "nt": 15}, INVALID)])
def test_store_refuses(call, args, code):
    rc, kernels, msg = call(store(**args))[0]
    assert rc == code and not kernels and msg.startswith("kvq_store")


def test_store_calls(call):
    few, many, host, same, none = call(store(), store(nt=16), store(pos=0, off=125), store(q=3, ldq=512),
                                       store(rot=0, rope=0))
    assert all(c[0] == 0 and len(c[1]) == 1 for c in (few, many, host, same, none))
    assert "k_kvq_storeI" in few[1][0] and "k_kvq_store_blocksI" in many[1][0]
    assert call(store(ns=0), store(nt=0, qkv=0, k=0)) == [(0, [], "")] * 2


def load(type=Q8, k=1, v=1, ns=2, kv=2, hd=64, ctx=128, pos=1, off=0, n=5, ko=1, vo=1):
    return ["load", type, k, v, ns, kv, hd, ctx, pos, off, n, ko, vo]


@pytest.mark.parametrize("args,code", [
    ({"type": 12}, UNSUPPORTED), ({"hd": 32}, UNSUPPORTED), ({"k": 0}, INVALID), ({"vo": 0}, INVALID), ({"k": 2}, INVALID),
    ({"vo": 2}, INVALID), ({"ns": -1}, INVALID), ({"kv": 0}, INVALID), ({"n": -1}, INVALID), ({"ctx": 65}, INVALID),
    ({"pos": 0, "off": 124}, INVALID), ({"pos": 0, "off": -1}, INVALID), ({"ns": 40000}, INVALID)])
def test_load_refuses(call, args, code):
    rc, kernels, msg = call(load(**args))[0]
    assert rc == code and not kernels and msg.startswith("kvq_load")


def test_load_calls(call):
    a, b, c = call(load(), load(n=16), load(v=0, vo=0, pos=0, off=123))
    assert all(x[0] == 0 and len(x[1]) == 1 for x in (a, b, c))
    assert "k_kvq_loadI" in a[1][0] and "k_kvq_load_blocksI" in b[1][0]
    assert call(load(n=0), load(k=0, v=0, ko=0, vo=0), load(ns=0)) == [(0, [], "")] * 3


def attn(type=Q8, q=1, ldq=None, ns=2, nt=3, h=4, kv=2, hd=64, pk=1, pv=1, pl=100, pc=128, k=1, v=1, ctx=128, pos=1, off=0,
         lim=128, o=1, ldo=None, work=1):
    return ["attn", type, q, h * hd if ldq is None else ldq, ns, nt, h, kv, hd, pk, pv, pl, pc, k, v, ctx, pos, off, lim, o,
            h * hd if ldo is None else ldo, work]


@pytest.mark.parametrize("args,code", [
    ({"type": 2}, UNSUPPORTED), ({"hd": 80}, UNSUPPORTED), ({"q": 0}, INVALID), ({"o": 0}, INVALID), ({"k": 0}, INVALID),
    ({"v": 0}, INVALID), ({"pk": 0}, INVALID), ({"pv": 0}, INVALID), ({"work": 0}, INVALID), ({"q": 2}, INVALID),
    ({"o": 2}, INVALID), ({"k": 2}, INVALID), ({"pv": 2}, INVALID), ({"work": 2}, INVALID), ({"ldq": 252}, INVALID),
    ({"ldo": 257}, INVALID), ({"ns": -1}, INVALID), ({"nt": -2}, INVALID), ({"h": 5}, INVALID), ({"kv": 0}, INVALID),
    ({"h": 0}, INVALID), ({"pl": 129}, INVALID), ({"pl": -1}, INVALID), ({"pc": 100}, INVALID), ({"ctx": 130, "lim": 100}, INVALID),
    ({"lim": 0}, INVALID), ({"lim": 129}, INVALID), ({"pos": 0, "off": 126}, INVALID), ({"pos": 0, "off": -1}, INVALID),
    ({"ns": 1 << 15, "nt": 1 << 15}, INVALID), ({"ns": 1 << 22, "nt": 1, "h": 32, "kv": 1}, INVALID), ({"nt": 1 << 25, "ctx": 0x7fffff00 - 192, "lim": 0x7fffff00 - 192}, INVALID)])
def test_attention_refuses(call, args, code):
    rc, kernels, msg = call(attn(**args))[0]
    assert rc == code and not kernels and msg.startswith("attn_kvq")


def test_attention_does_nothing_for_nothing(call):
    assert call(attn(ns=0), attn(nt=0), attn(ns=0, q=0, k=0)) == [(0, [], "")] * 3


def test_sizes(call):
    got = [c[0] for c in call(["bytes", F16, 3, 2, 128, 64], ["bytes", Q8, 3, 2, 128, 64], ["bytes", Q4, 1, 4, 64, 128],
                              ["bytes", 8, 1, 1, 64, 64], ["bytes", Q8, 1, 1, 100, 64], ["bytes", Q8, 1, 1, 64, 96],
                              ["bytes", Q8, 0, 1, 64, 64], ["bytes", Q8, 1, 0, 64, 64], ["bytes", Q8, 1, 1, 0, 64],
                              ["bytes", Q8, 64, 8, 1 << 20, 128],
                              ["bytes", F16, 0x7fffffff, 0x7fffffff, 128, 64])]
    # the last one's product passes 64 bits
    assert got == [3 * 2 * 128 * 128, 3 * 2 * 128 * 66, 4 * 64 * 68, 0, 0, 0, 0, 0, 0, 64 * 8 * (1 << 20) * 132, 0]
    # no workspace where one chunk holds all; none for shapes that a call would refuse
    got = [c[0] for c in call(["work", 1, 1, 14, 2, 64, 0, 300], ["work", 1, 1, 5, 2, 64, 0, 300], ["work", 1, 1, 4, 2, 96, 0, 300],
                              ["work", 2, 1, 4, 2, 64, 100, 64])]
    assert got[:3] == [0, 0, 0] and got[3] == 2 * 8 * (4 * 64 + 8)


def kernels_of(call, ty, hd, case):
    S, T, H, KV, P, starts, limit, ctx = case
    rc, kernels, msg = call(attn(ty, ns=S, nt=T, h=H, kv=KV, hd=hd, pk=int(P > 0), pv=int(P > 0), pl=P, pc=(P + 63) // 64 * 64,
                                 ctx=ctx, lim=limit or ctx))[0]
    assert rc == 0, msg
    return [re.sub(r"^_ZN3orc\d+|EEv.*$", "", k) for k in kernels]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ty", [F16, Q8, Q4])
def test_the_gpu_tests_reach_every_attention_kernel(call, ty, hd):
    """Row tiles of 16, 32, 64 (one and two key groups) and 128, the launches that mix two of them, both merges: for
    every type and head size, and all but the merges with tokens that see different keys."""
    import test_gpu_kvq as t

    def reached(cases):
        return {k.split("I", 1)[0] + " " + ",".join(re.findall(r"Li(\d+)", k)[2 if "merge" not in k else 1:])
                for case in cases for k in kernels_of(call, ty, hd, case)}

    main = {"k_attn_kvq 1", "k_attn_kvq 2", "k_attn_kvq_tile 1,1", "k_attn_kvq_tile 1,2", "k_attn_kvq_tile 2,1",
            "k_attn_kvq_both 1,1", "k_attn_kvq_both 1,2", "k_attn_kvq_both 2,1", "k_attn_kvq_both 2,2"}
    merges = {"k_attn_kvq_merge 1", "k_attn_kvq_merge 4"}
    assert reached(t.ATTENTIONS + t.LARGE) == main | merges
    assert reached(t.ODD) >= main
