"""The 4-bit K/V cache: its append, its values and its raw rows bit for bit
against the format's definition, attention over it against 64 bits, and what it
refuses."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import libllmcpu_amd as nh
from libllmcpu_amd import hip_rt
import q4_ref as ref


def rows_of(seed, n, d, spread=1.0):
    rng = np.random.default_rng(seed)
    return ((rng.standard_normal((n, d)) + rng.standard_normal((1, d))) * spread).astype(np.float32)


def filled(n_seq, kv_dim, rows, seed=1):
    """A cache with positions 0 .. n_seq - 1 appended, and their values."""
    k, v = rows_of(seed, n_seq, kv_dim), rows_of(seed + 1, n_seq, kv_dim)
    kv = nh.KVCache([rows], [kv_dim], q4=True)
    for p in range(0, n_seq, rows):
        m = min(rows, n_seq - p)
        kv.append_f32(0, p, k[p:p + m], v[p:p + m])
    return kv, ref.values(ref.quantise(k)), ref.values(ref.quantise(v))


# ---- without a GPU ---------------------------------------------------------------------

def test_create_refuses_rows_and_widths_off_the_block():
    lib = nh.load_library()
    for rows, dim in (([0], [64]), ([-32], [64]), ([100], [64]), ([64], [48]), ([64], [0]), ([64, 33], [64, 64])):
        h = C.c_void_p()
        n = len(rows)
        st = lib.nnc_hip_kv_create_q4(n, (C.c_int32 * n)(*rows), (C.c_int32 * n)(*dim), C.byref(h))
        assert st == nh.NncStatus.INVALID_ARGUMENT and not h.value, (rows, dim)
        assert b"32" in lib.nnc_hip_last_error()
    assert lib.nnc_hip_kv_create_q4(1, (C.c_int32 * 1)(64), (C.c_int32 * 1)(64), None) == nh.NncStatus.INVALID_ARGUMENT
    h = C.c_void_p()
    assert lib.nnc_hip_kv_create_q4(0, None, None, C.byref(h)) == nh.NncStatus.INVALID_ARGUMENT


def test_null_cache():
    lib = nh.load_library()
    assert lib.nnc_hip_kv_read_f32_device(None, 0, 0, 1, None, None) == nh.NncStatus.INVALID_ARGUMENT


def test_largest_values_stay_finite():
    """The bound behind the format's clamp: a block over the whole range ends on
    finite float16, and so does any other."""
    for lo, hi in ((-ref.Q4_MAX, ref.Q4_MAX), (-1e30, 1e30), (ref.Q4_MAX - 1, ref.Q4_MAX), (0, ref.Q4_MAX), (-3, ref.Q4_MAX)):
        x = np.linspace(lo, hi, 32, dtype=np.float64).astype(np.float32)[None]
        assert np.isfinite(ref.values(ref.quantise(x))).all(), (lo, hi)


# ---- the append ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,pos0,n", [
    (64, 32, 0, 1), (64, 32, 0, 64), (256, 128, 31, 2), (256, 1024, 250, 13), (96, 96, 7, 96), (96, 96, 1000, 95),
    (32, 64, 5, 32), (32, 64, 31, 1), (2048, 256, 1500, 1999), (8192, 512, 0, 8192), (64, 64, 2147483600, 40),
])
def test_append_and_values_bitwise(rows, dim, pos0, n):
    """Rows before and after are kept: the batch lands on a ring full of others."""
    print(f"append rows {rows} dim {dim} pos0 {pos0} n {n}", flush=True)
    old = [rows_of(s, rows, dim) for s in (5, 6)]
    new = [rows_of(s, n, dim, 3.0) for s in (7, 8)]
    at = (pos0 + np.arange(n, dtype=np.int64)) % rows
    want, raws = [], []
    for o, x in zip(old, new):
        qo, qx = ref.quantise(o), ref.quantise(x)
        w, r = ref.values(qo), ref.raw(qo)
        w[at], r[at] = ref.values(qx), ref.raw(qx)
        want.append(w)
        raws.append(r)
    with nh.KVCache([rows], [dim], q4=True) as kv:
        assert kv.nbytes == rows * dim * 2 * 5 // 8
        kv.append_f32(0, 0, *old)
        kv.append_f32(0, pos0, *new)
        got = kv.read_f32(0, 0, rows)
        got_raw = kv.read(0, 0, rows)
        part = kv.read_f32(0, rows // 3, rows // 2)
        part_raw = kv.read(0, rows // 3, rows // 2)
        for i in range(2):
            assert np.array_equal(got[i].astype(np.float64), want[i])
            assert np.array_equal(got_raw[i], raws[i])
            assert np.array_equal(part[i].astype(np.float64), want[i][rows // 3:rows // 3 + rows // 2])
            assert np.array_equal(part_raw[i], raws[i][rows // 3:rows // 3 + rows // 2])
        # the interchange rows, back in at another place
        kv.append(0, pos0 + 3, *(r[:n] for r in raws))
        at = (pos0 + 3 + np.arange(n, dtype=np.int64)) % rows
        back = kv.read(0, 0, rows)
        for i in range(2):
            w = raws[i].copy()
            w[at] = raws[i][:n]
            assert np.array_equal(back[i], w)


@pytest.mark.gpu
def test_append_of_unusual_elements():
    """Constant blocks, zeros, steps below float16's, the largest, infinities and
    NaN: bits of the definition, finite."""
    x = rows_of(3, 8, 64)
    x[0, :32], x[0, 32:] = 0, -0.0
    x[1, :] = 7.25
    x[2, :] *= 1e-9
    x[3, :] *= 1e-5
    x[4, :] *= 1e6
    x[5, 3], x[5, 40] = np.nan, np.inf
    x[6, :] = np.nan
    x[7, :32], x[7, 32:] = np.linspace(-1e30, 1e30, 32), np.linspace(60000, 70000, 32)
    with nh.KVCache([32], [64], q4=True) as kv:
        kv.append_f32(0, 0, x, x[::-1].copy())
        k, v = kv.read_f32(0, 0, 8)
    assert np.isfinite(k).all() and np.isfinite(v).all()
    want = ref.values(ref.quantise(x))
    assert np.array_equal(k.astype(np.float64), want) and np.array_equal(v[::-1].astype(np.float64), want)


@pytest.mark.gpu
def test_values_of_the_other_caches():
    for bf16 in (True, False):
        k, v = rows_of(1, 40, 24), rows_of(2, 40, 24)
        with nh.KVCache([48], [24], bf16=bf16) as kv:
            kv.append_f32(0, 0, k, v)
            got = kv.read_f32(0, 5, 30)
        for g, x in zip(got, (k, v)):
            want = nh.bf16_to_f32(nh.bf16_round(x)) if bf16 else x
            assert np.array_equal(g, want.reshape(x.shape)[5:35])


@pytest.mark.gpu
def test_refusals():
    lib = nh.load_library()
    with nh.KVCache([64], [80 * 2], q4=True) as kv:  # 2 heads of 80
        x = np.zeros((4, 160), np.float32)
        for pos0, n in ((-1, 1), (0, 65)):
            with pytest.raises(nh.NncError) as e:
                kv.append_f32(0, pos0, np.zeros((n, 160), np.float32), np.zeros((n, 160), np.float32))
            assert e.value.status == nh.NncStatus.INVALID_ARGUMENT
        with pytest.raises(nh.NncError) as e:
            kv.attend(0, x, pos0=0, n_head=2, n_kv=2, head_dim=80, scale=1.0)
        assert e.value.status == nh.NncStatus.UNSUPPORTED_MODEL and "4-bit" in e.value.message
        good = ref.raw(ref.quantise(x))
        for s, z in ((np.nan, 0), (np.inf, 0), (0, -np.inf), (4300, 1500), (-4300, -1500)):
            bad = good.copy()
            bad[2, 20:24] = np.array([s, z], np.float16).view(np.uint8)
            for k, v in ((bad, good), (good, bad)):
                with pytest.raises(nh.NncError) as e:
                    kv.append(0, 0, k, v)
                assert e.value.status == nh.NncStatus.INVALID_ARGUMENT and "row 2, block 1" in e.value.message
        d = hip_rt.malloc(4096)
        try:
            assert lib.nnc_hip_kv_append_f32_device(kv.handle, 0, 0, 1, d + 4, d) == nh.NncStatus.INVALID_ARGUMENT
            assert lib.nnc_hip_kv_read_f32_device(kv.handle, 0, 0, 1, d + 8, None) == nh.NncStatus.INVALID_ARGUMENT
            for row0, n in ((-1, 1), (0, 65), (64, 1), (2147483647, 1)):
                assert lib.nnc_hip_kv_read_f32_device(kv.handle, 0, row0, n, d, None) == nh.NncStatus.INVALID_ARGUMENT
            assert lib.nnc_hip_kv_read_f32_device(kv.handle, 0, 64, 0, d, None) == nh.NncStatus.OK
        finally:
            hip_rt.free(d)


# ---- attention ------------------------------------------------------------------------------

CASES = [  # n_head, n_kv, head_dim, rows, n_seq, pos0, n_tok, window, causal
    (1, 1, 32, 32, 1, 0, 1, 0, True),
    (4, 1, 256, 1024, 1000, 999, 1, 0, True),
    (32, 8, 128, 4096, 3001, 3000, 1, 0, True),
    (32, 8, 64, 4096, 4096, 4095, 1, 0, True),
    (6, 2, 96, 512, 500, 487, 13, 0, True),
    (14, 2, 64, 640, 613, 600, 13, 100, True),
    (16, 1, 128, 256, 200, 199, 1, 0, True),
    (3, 1, 256, 512, 400, 0, 16, 0, False),
    (2, 2, 512, 256, 130, 128, 2, 0, True),
    (16, 16, 512, 96, 70, 64, 6, 33, True),
    (4, 4, 192, 256, 250, 240, 10, 64, False),
    (8, 4, 256, 768, 5000, 4990, 10, 512, True),  # a wrapped ring
    (32, 8, 128, 512, 300, 17, 283, 0, True),
    (4, 1, 256, 1024, 1500, 1100, 400, 256, True),  # a wrapped ring
    (5, 5, 64, 256, 200, 0, 200, 0, False),
    (12, 4, 128, 256, 180, 0, 180, 40, False),
    (32, 8, 64, 256, 33, 0, 33, 0, True),
    (7, 1, 96, 256, 250, 33, 217, 0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,hd,rows,n_seq,pos0,n_tok,window,causal", CASES)
def test_attention(n_head, n_kv, hd, rows, n_seq, pos0, n_tok, window, causal):
    print(f"attend {n_head}/{n_kv}/{hd} rows {rows} n_seq {n_seq} tokens {pos0}+{n_tok} window {window}", flush=True)
    shape = dict(window=window, causal=causal, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    q = rows_of(9, n_tok, n_head * hd)
    kv, k, v = filled(n_seq, n_kv * hd, rows)
    with kv:
        got = kv.attend(0, q, pos0=pos0, n_seq=n_seq, **shape)
        gate = rows_of(10, n_tok, n_head * hd)
        gated = kv.attend(0, q, pos0=pos0, n_seq=n_seq, gate=gate, **shape)
    want, bound, _ = ref.attend(q, k, v, pos0=pos0, n_seq=n_seq, **shape)
    d = np.abs(got - want)
    assert (d <= bound).all(), f"{d.max():.3g}, {(d / bound).max():.3g} of the bound"
    sig = 1 / (1 + np.exp(-gate.astype(np.float64)))
    assert (np.abs(gated - want * sig) <= bound * sig + 2.0**-21 * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,hd,n_seq,window", [(32, 8, 128, 5000, 0), (4, 1, 256, 900, 512), (6, 2, 96, 700, 0),
                                                         (14, 2, 64, 2100, 0), (16, 1, 32, 300, 0)])
def test_batch_bits(n_head, n_kv, hd, n_seq, window):
    """Every token of a session batch, and of any batch in exact mode, has the bits
    of its one-token call."""
    shape = dict(window=window, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    kv, _, _ = filled(n_seq, n_kv * hd, (n_seq + 31) // 32 * 32)
    with kv:
        for n, exact in ((2, False), (7, False), (16, False), (40, True)):
            kv.set_exact_batches(exact)
            q = rows_of(n, n, n_head * hd)
            p0 = n_seq - n
            batch = kv.attend(0, q, pos0=p0, n_seq=n_seq, **shape)
            for t in range(n):
                one = kv.attend(0, q[t:t + 1], pos0=p0 + t, n_seq=n_seq, **shape)
                assert np.array_equal(one[0], batch[t]), (n, t)


@pytest.mark.gpu
def test_ring_is_a_full_buffer():
    shape = dict(window=200, n_head=8, n_kv=2, head_dim=128, scale=0.1)
    full, _, _ = filled(1300, 256, 1312)
    ring, _, _ = filled(1300, 256, 256)
    q = rows_of(2, 16, 1024)
    with full, ring:
        assert np.array_equal(full.attend(0, q, pos0=1284, **shape), ring.attend(0, q, pos0=1284, **shape))


@pytest.mark.gpu
def test_tokens_that_see_nothing_and_large_scores():
    hd = 64
    kv, k, v = filled(300, 2 * hd, 320)
    with kv:
        # a drafter at position 5 with a window of 2 over the first 3 keys: token 0 sees none of them
        shape = dict(window=2, causal=True, n_head=4, n_kv=2, head_dim=hd, scale=0.125)
        q = rows_of(4, 3, 4 * hd)
        got = kv.attend(0, q, pos0=3, n_seq=3, **shape)
        want, bound, _ = ref.attend(q, k, v, pos0=3, n_seq=3, **shape)
        assert not got[1:].any() and (np.abs(got - want) <= bound).all()
        # scores of thousands, of both signs, and none at all
        shape = dict(window=0, causal=True, n_head=4, n_kv=2, head_dim=hd, scale=0.125)
        for f in (3000.0, 1e-30, 0.0):
            q = rows_of(5, 2, 4 * hd) * np.float32(f)
            got = kv.attend(0, q, pos0=298, **shape)
            want, bound, _ = ref.attend(q, k, v, pos0=298, n_seq=300, **shape)
            assert (np.abs(got - want) <= bound).all(), f
        # one token's q is NaN, and one infinite: the others' rows are untouched
        q = rows_of(6, 4, 4 * hd)
        clean = kv.attend(0, q, pos0=296, **shape)
        q[1, 3], q[3, 70] = np.nan, np.inf
        got = kv.attend(0, q, pos0=296, **shape)
        hit = np.zeros_like(got, bool)
        hit[1, :hd], hit[3, hd:2 * hd] = True, True
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.gpu
def test_long_cache_past_32_bits():
    """Records past 4 GiB: the last rows of a buffer of 5.4 GB."""
    rows, dim = 131072 * 16, 4096
    with nh.KVCache([rows], [dim], q4=True) as kv:
        assert kv.nbytes > 1 << 32
        n = 400
        k, v = rows_of(1, n, dim), rows_of(2, n, dim)
        kv.append_f32(0, rows - n, k, v)
        got = kv.read_f32(0, rows - n, n)
        kq, vq = ref.values(ref.quantise(k)), ref.values(ref.quantise(v))
        assert np.array_equal(got[0].astype(np.float64), kq) and np.array_equal(got[1].astype(np.float64), vq)
        shape = dict(window=150, causal=True, n_head=32, n_kv=32, head_dim=128, scale=0.09)
        for m in (1, 20):
            q = rows_of(3, m, dim)
            out = kv.attend(0, q, pos0=rows - m, **shape)
            want, bound, _ = ref.attend(q, kq, vq, pos0=n - m, n_seq=n, **shape)
            assert (np.abs(out - want) <= bound).all()


@pytest.mark.gpu
def test_prep_append_then_decode():
    """The pre-attention step into a 4-bit cache is the same step into an F32 one,
    quantised; and attention reads what it wrote."""
    hd, n_head, n_kv, n = 128, 8, 2, 45
    prep = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, q_gamma=1 + rows_of(1, 1, hd)[0] / 8, k_gamma=1 + rows_of(2, 1, hd)[0] / 8,
                n_rot=hd, base=1e6)
    q, k, v = rows_of(3, n, n_head * hd), rows_of(4, n, n_kv * hd), rows_of(5, n, n_kv * hd)
    with nh.KVCache([64], [n_kv * hd], q4=True) as kv, nh.KVCache([64], [n_kv * hd], bf16=False) as f32:
        q4 = kv.prep_append(0, q, k, v, pos0=40, **prep)
        qf = f32.prep_append(0, q, k, v, pos0=40, **prep)
        assert np.array_equal(q4, qf)
        for a, b in zip(kv.read_f32(0, 0, 64), f32.read_f32(0, 0, 64)):
            assert np.array_equal(a.astype(np.float64), ref.values(ref.quantise(b)))


@pytest.mark.gpu
@pytest.mark.parametrize("n_tok", [1, 5, 100])
def test_captured_and_noalloc(n_tok):
    """A decode step and batches in a HIP graph, replayed between eager work on the
    same cache, and the entry point that allocates nothing."""
    hd, n_head, n_kv, n_seq = 128, 16, 4, 700
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=0.09)
    kv, _, _ = filled(n_seq, n_kv * hd, 1024)
    q = [rows_of(20 + i, n_tok, n_head * hd) for i in range(4)]
    nb = q[0].nbytes
    with kv:
        want = [kv.attend(0, x, pos0=n_seq - n_tok, **shape) for x in q]
        dq, do = hip_rt.malloc(nb), hip_rt.malloc(nb)
        try:
            def call():
                kv.attend_device(0, dq, do, n_tok=n_tok, pos0=n_seq - n_tok, **shape)

            graph = hip_rt.Graph(kv.stream, call)
            for x, w in zip(q, want):
                hip_rt.to_device(dq, x)
                graph.launch(kv.stream)
                kv.sync()
                assert np.array_equal(hip_rt.to_host(np.empty_like(x), do), w)
                kv.attend(0, rows_of(1, 9, n_head * hd), pos0=n_seq - 9, **shape)
            graph.close()
            kv.attend_device_noalloc(0, dq, do, n_tok=n_tok, pos0=n_seq - n_tok, **shape)
            kv.sync()
            assert np.array_equal(hip_rt.to_host(np.empty_like(q[3]), do), want[3])
        finally:
            hip_rt.free(dq)
            hip_rt.free(do)


@pytest.mark.gpu
def test_two_caches_at_once():
    """Two sessions' caches in use together, each on its own stream, issued in turn."""
    hd, shape = 64, dict(n_head=8, n_kv=2, head_dim=64, scale=0.125)
    both = [filled(n, 2 * hd, 1024, seed=s) for n, s in ((1000, 1), (640, 11))]
    q = [rows_of(30 + i, 1, 8 * hd) for i in range(2)]
    dev = [hip_rt.malloc(8 * hd * 4) for _ in range(4)]
    try:
        want = [kv.attend(0, x, pos0=n - 1, **shape) for (kv, _, _), x, n in zip(both, q, (1000, 640))]
        for d, x in zip(dev, q):
            hip_rt.to_device(d, x)
        for _ in range(20):
            for i, n in enumerate((1000, 640)):
                both[i][0].attend_device(0, dev[i], dev[2 + i], n_tok=1, pos0=n - 1, **shape)
        for i in range(2):
            both[i][0].sync()
            assert np.array_equal(hip_rt.to_host(np.empty_like(q[i]), dev[2 + i]), want[i])
    finally:
        for kv, _, _ in both:
            kv.close()
        for d in dev:
            hip_rt.free(d)


# ---- few tokens over many keys: their keys shared among work-groups ---------------------

SHARED = [  # n_head, n_kv, head_dim, rows, n_seq, pos0, n_tok, window, causal
    (4, 1, 256, 4096, 4000, 3980, 20, 0, True),
    (32, 8, 128, 2560, 2500, 2460, 40, 0, True),
    (14, 2, 64, 2048, 1901, 1871, 30, 0, True),
    (6, 2, 96, 2304, 6000, 5950, 50, 2100, True),  # a wrapped ring
    (3, 1, 192, 2048, 2000, 100, 25, 0, False),
    (2, 1, 32, 4096, 3333, 3300, 17, 3001, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,hd,rows,n_seq,pos0,n_tok,window,causal", SHARED)
def test_few_tokens_over_many_keys(n_head, n_kv, hd, rows, n_seq, pos0, n_tok, window, causal):
    """Against 64 bits, gated too; the entry point that allocates nothing and a
    graph captured after the first call give the same bits, one captured before
    it is within the same bound."""
    print(f"few over many {n_head}/{n_kv}/{hd} rows {rows} n_seq {n_seq} tokens {pos0}+{n_tok} window {window}", flush=True)
    shape = dict(window=window, causal=causal, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    q, gate = rows_of(9, n_tok, n_head * hd), rows_of(10, n_tok, n_head * hd)
    kv, k, v = filled(n_seq, n_kv * hd, rows)
    want, bound, _ = ref.attend(q, k, v, pos0=pos0, n_seq=n_seq, **shape)
    dq, do = hip_rt.malloc(q.nbytes), hip_rt.malloc(q.nbytes)
    try:
        with kv:
            hip_rt.to_device(dq, q)

            def call(noalloc=False):
                f = kv.attend_device_noalloc if noalloc else kv.attend_device
                f(0, dq, do, n_tok=n_tok, pos0=pos0, n_seq=n_seq, **shape)

            def out():
                kv.sync()
                return hip_rt.to_host(np.empty_like(q), do)

            early = hip_rt.Graph(kv.stream, call)
            early.launch(kv.stream)
            assert (np.abs(out() - want) <= bound).all()
            call()
            got = out()
            assert (np.abs(got - want) <= bound).all()
            late = hip_rt.Graph(kv.stream, call)
            for _ in range(3):
                late.launch(kv.stream)
                assert np.array_equal(out(), got)
                kv.attend(0, q[:1], pos0=pos0, n_seq=n_seq, **shape)
                early.launch(kv.stream)
                assert (np.abs(out() - want) <= bound).all()
            call(noalloc=True)
            assert np.array_equal(out(), got)
            gated = kv.attend(0, q, pos0=pos0, n_seq=n_seq, gate=gate, **shape)
            early.close()
            late.close()
    finally:
        hip_rt.free(dq)
        hip_rt.free(do)
    sig = 1 / (1 + np.exp(-gate.astype(np.float64)))
    assert (np.abs(gated - want * sig) <= bound * sig + 2.0**-21 * np.abs(want)).all()


@pytest.mark.gpu
def test_positions_past_the_limit():
    """Rings keep any position up to 2^30; past it the attend calls refuse."""
    far = (1 << 30) - 40
    shape = dict(window=100, causal=True, n_head=2, n_kv=1, head_dim=64, scale=0.125)
    k, v, q = rows_of(1, 256, 64), rows_of(2, 256, 64), rows_of(3, 30, 128)
    with nh.KVCache([256], [64], q4=True) as kv:
        kv.append_f32(0, far - 226, k, v)  # positions far - 226 .. far + 29
        for n in (30, 3, 1):
            got = kv.attend(0, q[:n], pos0=far + 30 - n, n_seq=far + 30, **shape)
            want, bound, _ = ref.attend(q[:n], ref.values(ref.quantise(k)), ref.values(ref.quantise(v)), pos0=256 - n, n_seq=256, **shape)
            assert (np.abs(got - want) <= bound).all()
        for bad in (dict(pos0=far + 30), dict(pos0=far, n_seq=(1 << 30) + 1), dict(pos0=2**31 - 31), dict(pos0=far, window=2**31 - 1, causal=False)):
            with pytest.raises(nh.NncError) as e:
                kv.attend(0, q, **{**shape, "n_seq": far + 30, **bad})
            assert e.value.status == nh.NncStatus.INVALID_ARGUMENT


CORNERS = [  # n_head, n_kv, head_dim, rows, n_seq, pos0, n_tok, window, causal
    (16, 1, 512, 1024, 900, 899, 1, 0, True),
    (16, 1, 512, 1024, 900, 862, 38, 0, True),
    (16, 1, 192, 2048, 1999, 1998, 1, 0, True),
    (32, 2, 128, 4096, 4000, 3984, 16, 0, True),  # 256 pairs a KV head
    (11, 1, 32, 8192, 8000, 7999, 1, 0, True),
    (33, 11, 32, 96, 90, 80, 10, 1, True),  # every token its own key alone
    (8, 2, 64, 512, 300, 400, 3, 0, True),  # positions past the last key
    (8, 2, 64, 512, 300, 400, 30, 0, True),
    (8, 2, 64, 512, 300, 280, 60, 25, True),  # the last tokens see nothing
    (8, 2, 96, 512, 300, 285, 14, 7, False),
    (1, 1, 256, 64, 40, 0, 40, 2, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,hd,rows,n_seq,pos0,n_tok,window,causal", CORNERS)
def test_corners(n_head, n_kv, hd, rows, n_seq, pos0, n_tok, window, causal):
    """The largest groups and heads, the narrowest windows, positions past the last
    key; in exact mode every token has its one-token bits."""
    print(f"corner {n_head}/{n_kv}/{hd} rows {rows} n_seq {n_seq} tokens {pos0}+{n_tok} window {window}", flush=True)
    shape = dict(n_seq=n_seq, window=window, causal=causal, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    q = rows_of(9, n_tok, n_head * hd)
    kv, k, v = filled(n_seq, n_kv * hd, rows)
    with kv:
        got = kv.attend(0, q, pos0=pos0, **shape)
        want, bound, _ = ref.attend(q, k, v, pos0=pos0, **shape)
        assert (np.abs(got - want) <= bound).all()
        kv.set_exact_batches(True)
        exact = kv.attend(0, q, pos0=pos0, **shape)
        for t in sorted({0, n_tok // 2, n_tok - 1}):
            assert np.array_equal(exact[t:t + 1], kv.attend(0, q[t:t + 1], pos0=pos0 + t, **shape)), t


@pytest.mark.gpu
@pytest.mark.parametrize("n_head,n_kv,hd,n_seq,window", [
    (32, 8, 128, 500, 0), (32, 8, 128, 2000, 0), (32, 8, 128, 9000, 0), (32, 8, 64, 2000, 300), (4, 1, 256, 1000, 0), (4, 1, 256, 8000, 0),
    (8, 4, 256, 3000, 0), (12, 4, 192, 700, 0), (16, 4, 32, 900, 0), (12, 6, 96, 400, 0), (6, 3, 512, 600, 0)])
def test_batch_bits_whatever_the_kernel(n_head, n_kv, hd, n_seq, window):
    """Batches of as many (token, head) pairs as one wavefront, two, a work-group per
    tile or the kernel for many take."""
    shape = dict(n_seq=n_seq, window=window, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    kv, k, v = filled(n_seq, n_kv * hd, (n_seq + 31) // 32 * 32)
    q = rows_of(3, 16, n_head * hd)
    with kv:
        one = [kv.attend(0, q[t:t + 1], pos0=n_seq - 16 + t, **shape)[0] for t in range(16)]
        want, bound, _ = ref.attend(q, k, v, pos0=n_seq - 16, causal=True, **shape)
        assert (np.abs(np.array(one) - want) <= bound).all()
        for a, b in ((0, 16), (13, 16), (9, 13), (3, 8), (10, 16), (0, 8), (1, 14), (14, 16)):
            print(f"bits {n_head}/{n_kv}/{hd} n_seq {n_seq} tokens {a} .. {b}", flush=True)
            assert np.array_equal(kv.attend(0, q[a:b], pos0=n_seq - 16 + a, **shape), np.array(one[a:b])), (a, b)
