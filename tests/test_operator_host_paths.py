"""What the host code of packed attention and of the 4-bit cache launches, without
a GPU, over a HIP runtime of the test's own (hip_stub_flash.cpp). Each check runs
in a process of its own, since a process binds one runtime."""
from __future__ import annotations

import ctypes as C
import random
import subprocess
import sys
from pathlib import Path

import pytest

HERE = Path(__file__).resolve()
CHECKS = {}
MIB = 1 << 20
Q, K, V, OUT = (x << 20 for x in (1, 2, 3, 4))  # (addresses are not read: nothing runs)


def check(fn):
    CHECKS[fn.__name__] = fn
    return fn


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = tmp_path_factory.mktemp("hip_stub_flash") / "libhip_stub_flash.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-DNNC_STUB_SYMBOL_BYTES={32 * MIB}", str(HERE.parent / "hip_stub_flash.cpp"), "-o", str(so)], check=True)
    return so


class Runtime:
    def __init__(self, so: str):
        self.lib = C.CDLL(so, mode=C.RTLD_GLOBAL)  # before libnnc_hip.so is loaded
        for f in ("stub_flash_part", "stub_symbol"):
            getattr(self.lib, f).restype = C.c_void_p
        self.lib.stub_name.restype = C.c_char_p
        self.lib.stub_bytes_left.restype = C.c_size_t
        self.lib.stub_bytes_left.argtypes = [C.c_void_p]

    def clear(self):
        self.lib.stub_flash_clear()

    def launches(self):
        got = []
        for i in range(self.lib.stub_launches()):
            v = (C.c_longlong * 9)()
            self.lib.stub_flash(i, v)
            l = dict(zip(("kind", "device", "grid", "block", "n", "key_groups", "n_head", "n_kv", "head_dim"), v),
                     name=self.lib.stub_name(i).decode(), part=self.lib.stub_flash_part(i), seqs=[])
            for s in range(l["n"]):
                w = (C.c_int * 5)()
                self.lib.stub_flash_seq(i, s, w)
                l["seqs"].append(dict(zip(("start", "len", "tile", "split", "part"), w)))
            got.append(l)
        return got


def tiles_fit(rt, launches, what):
    """Every launch's table is its grid, a work-group a tile and split; partials of
    shared tiles are apart and inside their allocation, and merged by the launch behind."""
    for i, l in enumerate(launches):
        assert l["kind"] in (1, 2) and l["grid"] * l["block"] < 1 << 32, what
        if l["kind"] == 2:
            continue
        rows = 64 if l["head_dim"] > 128 and l["key_groups"] == 2 else 128
        group, at, part, shared = l["n_head"] // l["n_kv"], 0, 0, []
        for s in l["seqs"]:
            assert s["len"] > 0 and s["tile"] == at and s["split"] >= 1, what
            at += -(-s["len"] * group // rows) * s["split"]
            if s["split"] > 1:
                assert s["part"] == part, what
                part += s["len"] * l["n_head"] * s["split"]
                shared.append(s)
        assert l["grid"] == at * l["n_kv"], what
        need = part * (l["head_dim"] + 4) * 4
        assert need <= 32 * MIB, what
        if not shared:
            assert i + 1 == len(launches) or launches[i + 1]["kind"] == 1, what
            continue
        left = rt.lib.stub_bytes_left(l["part"])
        if l["part"] == rt.lib.stub_symbol():
            left = 32 * MIB
        assert need <= left, what
        m = launches[i + 1]
        assert m["kind"] == 2 and m["part"] == l["part"], what
        assert [(s["start"], s["len"], s["split"], s["part"]) for s in m["seqs"]] == \
            [(s["start"], s["len"], s["split"], s["part"]) for s in shared], what
        here = 256 // (l["head_dim"] // 4)
        at = 0
        for s in m["seqs"]:
            assert s["tile"] == at, what
            at += -(-s["len"] * l["n_head"] // here)
        assert m["grid"] == at, what


@check
def packed_tables(rt, nh):
    rng = random.Random(5)
    shapes = [(1, 1, 8), (4, 1, 256), (32, 8, 128), (14, 2, 64), (6, 2, 96), (64, 1, 16), (3, 1, 200), (8, 8, 64)]
    lens = [[1], [0], [5000, 1, 0, 3], [700] * 130, [3000, 2900, 10], [9, 4, 70000]]
    lens += [[int(2 ** rng.uniform(0, 12)) for _ in range(rng.randrange(1, 90))] for _ in range(12)]
    for n_head, n_kv, hd in shapes:
        for ls in lens:
            for bf16, window, causal in ((True, 0, True), (False, 300, False), (True, 0, False), (False, 64, True)):
                what = (n_head, n_kv, hd, len(ls), max(ls), bf16, window, causal)
                starts = [7]
                for n in ls:
                    starts.append(starts[-1] + n)
                with nh.KVCache([32], [32]) as kv:
                    for _ in range(2):
                        rt.clear()
                        kv.attend_packed_device(Q, K, V, OUT, starts=starts, bf16=bf16, window=window, causal=causal, n_head=n_head,
                                                n_kv=n_kv, head_dim=hd, scale=0.1)
                        got = rt.launches()
                        tiles_fit(rt, got, what)
                        listed = sorted((s["start"], s["len"]) for l in got if l["kind"] == 1 for s in l["seqs"])
                        assert listed == sorted((a, b - a) for a, b in zip(starts, starts[1:]) if b > a), what


@check
def batches_over_four_bits(rt, nh):
    for n_head, n_kv, hd in ((4, 1, 256), (32, 8, 128), (2, 1, 32), (16, 1, 192)):
        for n_tok, n_seq, window in ((17, 17, 0), (20, 8000, 0), (512, 4096, 0), (900, 5000, 0), (40, 6000, 700), (3000, 8000, 0)):
            what = (n_head, n_kv, hd, n_tok, n_seq, window)
            with nh.KVCache([8192], [n_kv * hd], q4=True) as kv:
                def call(f):
                    rt.clear()
                    f(0, Q, OUT, n_tok=n_tok, pos0=n_seq - n_tok, n_seq=n_seq, window=window, causal=True, n_head=n_head, n_kv=n_kv,
                      head_dim=hd, scale=0.1)
                    tiles_fit(rt, rt.launches(), what)
                    return [[(s["len"], s["split"], s["part"]) for s in l["seqs"]] for l in rt.launches()]

                first = call(kv.attend_device)
                assert call(kv.attend_device_noalloc) == first, what  # the same splits: the same bits


@check
def captured_before_and_after_the_scratch(rt, nh):
    """A capture allocates nothing: without scratch nothing is shared, with too little
    as much as fits, and afterwards what an eager call shares."""
    def packed(kv, n=4000):
        kv.attend_packed_device(Q, K, V, OUT, starts=[0, n], bf16=True, n_head=2, n_kv=1, head_dim=64, scale=0.1)

    def over4(kv, n=20):
        kv.attend_device(0, Q, OUT, n_tok=n, pos0=8000 - n, n_seq=8000, window=0, causal=True, n_head=2, n_kv=1, head_dim=64, scale=0.1)

    for call in (packed, over4):
        with nh.KVCache([8192], [64], q4=True) as kv:
            def captured():
                rt.clear()
                rt.lib.stub_capture(1)
                call(kv)
                rt.lib.stub_capture(0)
                assert not rt.lib.stub_capture_invalid(), call.__name__
                got = rt.launches()
                tiles_fit(rt, got, call.__name__)
                return max(s["split"] for l in got for s in l["seqs"])

            assert captured() == 1
            kv.attend_device(0, Q, OUT, n_tok=1, pos0=2047, n_seq=2048, window=0, causal=True, n_head=2, n_kv=1, head_dim=64, scale=0.1)
            some = captured()
            rt.clear()
            call(kv)
            eager = max(s["split"] for l in rt.launches() for s in l["seqs"])
            assert 1 <= some <= eager and eager > 1 and captured() == eager


@check
def on_the_cache_s_device(rt, nh):
    """With another device current every launch and allocation is on the cache's, and
    the caller's is current afterwards; after refusals too."""
    import numpy as np

    rt.lib.hipSetDevice(1)
    kv = nh.KVCache([4096], [64], q4=True)
    rt.lib.hipSetDevice(0)
    shape = dict(n_head=2, n_kv=1, head_dim=64, scale=0.1)
    x, q = np.zeros((40, 64), np.float32), np.zeros((40, 128), np.float32)
    raw = np.zeros((40, 40), np.uint8)
    calls = {
        "append": lambda: kv.append(0, 0, raw, raw),
        "append_f32": lambda: kv.append_f32(0, 0, x, x),
        "append_f32_device": lambda: kv.append_f32_device(0, K, V, pos0=0, n_tok=9),
        "read": lambda: kv.read(0, 0, 40),
        "read_f32_device": lambda: kv.read_f32_device(0, 0, 40, K, V),
        "attend": lambda: kv.attend(0, q, pos0=0, n_seq=40, **shape),
        "attend_device": lambda: kv.attend_device(0, Q, OUT, n_tok=20, pos0=3980, n_seq=4000, window=0, causal=True, **shape),
        "attend_device_noalloc": lambda: kv.attend_device_noalloc(0, Q, OUT, n_tok=1, pos0=3999, n_seq=4000, window=0, causal=True, **shape),
        "attend_packed": lambda: kv.attend_packed_device(Q, K, V, OUT, starts=[0, 5000], bf16=False, **shape),
    }
    for name, call in calls.items():
        rt.clear()
        call()
        got = rt.launches()
        assert got and all(l["device"] == 1 for l in got), name
        assert rt.lib.stub_malloc_devices() in (0, 2) and rt.lib.stub_device() == 0, name
    with pytest.raises(nh.NncError):
        kv.attend_packed_device(Q, K, V, OUT, starts=[0, 5000], bf16=False, **{**shape, "head_dim": 60})
    with pytest.raises(nh.NncError):
        kv.read_f32_device(0, 4090, 40, K, V)
    assert rt.lib.stub_device() == 0
    kv.close()


@check
def refusals_launch_nothing(rt, nh):
    ok = dict(q_stride=256, k_stride=128, v_stride=128, out_stride=256, starts=[0, 9, 20], bf16=True, n_head=4, n_kv=2, head_dim=64, scale=0.1)
    with nh.KVCache([64], [64], q4=True) as kv:
        rt.clear()
        for change in (dict(starts=[0, 9, 8]), dict(starts=[-1, 9]), dict(window=-1), dict(n_head=5), dict(n_kv=0), dict(head_dim=4),
                       dict(head_dim=264, q_stride=4096, k_stride=4096, v_stride=4096, out_stride=4096), dict(q_stride=248), dict(v_stride=132),
                       dict(k_stride=1 << 23), dict(starts=[0, 3, (1 << 27)]), dict(starts=[])):
            with pytest.raises(nh.NncError):
                kv.attend_packed_device(Q, K, V, OUT, **{**ok, **change})
        for a in ((Q + 8, K, V, OUT), (Q, K, V, K), (Q, K, V, V), (0, K, V, OUT), (Q, K, V, 0), (Q, K + 4, V, OUT)):
            with pytest.raises(nh.NncError):
                kv.attend_packed_device(*a, **ok)
        one = dict(n_tok=1, pos0=9, n_seq=10, window=0, causal=True, n_head=2, n_kv=1, head_dim=64, scale=0.1)
        for change in (dict(head_dim=32), dict(n_seq=(1 << 30) + 1), dict(pos0=1 << 30), dict(n_tok=0), dict(n_seq=200, pos0=150),
                       dict(window=(1 << 30) + 1), dict(n_head=34)):
            with pytest.raises(nh.NncError):
                kv.attend_device(0, Q, OUT, **{**one, **change})
        for row0, n in ((-1, 4), (0, 65), (64, 1), (0, -1)):
            with pytest.raises(nh.NncError):
                kv.read_f32_device(0, row0, n, K, V)
        with pytest.raises(nh.NncError):
            kv.append_f32_device(0, K + 4, V, pos0=0, n_tok=2)
        with pytest.raises(nh.NncError):
            kv.append_f32_device(0, K, V, pos0=0, n_tok=65)
        assert not rt.launches()


@pytest.mark.parametrize("name", sorted(CHECKS))
def test_operator_host_path(stub, name):
    r = subprocess.run([sys.executable, str(HERE), str(stub), name], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


if __name__ == "__main__":
    rt = Runtime(sys.argv[1])
    sys.path.insert(0, str(HERE.parents[1]))
    import libllmcpu_amd

    libllmcpu_amd.set_log_callback(lambda level, msg: None)
    CHECKS[sys.argv[2]](rt, libllmcpu_amd)
