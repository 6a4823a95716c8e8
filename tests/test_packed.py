"""Attention over several whole sequences laid end to end, against 64 bits: both
element types, head shapes, masks, strides, elements that are infinite or NaN,
what is refused, and together with the 4-bit cache as a server would use them."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import libllmcpu_amd as nh
from libllmcpu_amd import hip_rt
import q4_ref as ref


def rows_of(seed, n, d):
    return np.random.default_rng(seed).standard_normal((n, d)).astype(np.float32)


def typed(x, bf16):
    """(what the library takes, its values)"""
    if not bf16:
        return x, x.astype(np.float64)
    b = nh.bf16_round(x).reshape(x.shape)
    return b, nh.bf16_to_f32(b).astype(np.float64)


def as_values(x):
    return (nh.bf16_to_f32(x) if x.dtype == np.uint16 else x).astype(np.float64).reshape(x.shape)


def expected(q, k, v, starts, bf16, **shape):
    """(out, bound). Beyond q4_ref.attend's bound, F32: K and V have 22 bits too and
    lo x lo products are left out (2^-22 each: 2^-21 of a score's sum and of a
    value, within another 2^-20 of the largest |V|). BF16: a weight is off by 2^-8
    at most, so an output by 2^-8 of the mean |V|, and its own rounding."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for a, b in zip(starts, starts[1:]):
        if a == b:
            continue
        o, d, spread = ref.attend(q[a:b], k[a:b], v[a:b], pos0=0, n_seq=b - a, **shape)
        out[a:b] = o
        bound[a:b] = d + 2.0**-8 * (spread + np.abs(o)) if bf16 else d + 2.0**-20 * np.abs(v[a:b]).max()
    return out, bound


SHAPES = [(1, 1, 8), (4, 2, 64), (32, 8, 128), (6, 2, 96), (14, 2, 64), (3, 1, 256), (5, 5, 40), (9, 3, 200), (16, 1, 128)]
LENS = [[1], [2, 0, 1, 31, 32, 33], [130, 64, 65], [0, 257, 3, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("window,causal", [(0, True), (20, True), (0, False), (51, False)])
@pytest.mark.parametrize("n_head,n_kv,hd", SHAPES)
def test_packed(n_head, n_kv, hd, window, causal, bf16):
    shape = dict(window=window, causal=causal, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    with nh.KVCache([32], [32]) as kv:
        for lens in LENS:
            print(f"packed {n_head}/{n_kv}/{hd} window {window} causal {causal} bf16 {bf16} lens {lens}", flush=True)
            pad = 3  # rows before and after the sequences
            starts = [pad]
            for n in lens:
                starts.append(starts[-1] + n)
            total = starts[-1] + 2
            (q, q64), (k, k64), (v, v64) = (typed(rows_of(s, total, h * hd), bf16) for s, h in ((1, n_head), (2, n_kv), (3, n_kv)))
            got = kv.attend_packed(q, k, v, starts=starts, **shape)
            want, bound = expected(q64, k64, v64, starts, bf16, **shape)
            assert not got[:pad].any() and not got[starts[-1]:].any()
            d = np.abs(as_values(got) - want)
            assert (d <= bound).all(), f"{lens}: {d.max():.3g}, {(d / np.maximum(bound, 1e-30)).max():.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
def test_long_sequence_and_many_short_ones(bf16):
    """More sequences than one launch takes, one of them long."""
    rng = np.random.default_rng(3)
    lens = [int(n) for n in rng.integers(0, 9, 150)]
    lens[70] = 1500
    starts = [0, *np.cumsum(lens).tolist()]
    shape = dict(window=0, causal=True, n_head=4, n_kv=2, head_dim=64, scale=0.125)
    (q, q64), (k, k64), (v, v64) = (typed(rows_of(s, starts[-1], h * 64), bf16) for s, h in ((1, 4), (2, 2), (3, 2)))
    with nh.KVCache([32], [32]) as kv:
        got = kv.attend_packed(q, k, v, starts=starts, **shape)
    want, bound = expected(q64, k64, v64, starts, bf16, **shape)
    assert (np.abs(as_values(got) - want) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
def test_strides_and_in_place(bf16):
    """q, k and v as columns of one buffer, out over q; what lies between the columns
    and outside the sequences stays as it was. Every sequence has the bits of its
    call alone."""
    n_head, n_kv, hd, n = 6, 2, 72, 90
    qd, kd = n_head * hd, n_kv * hd
    size = 2 if bf16 else 4
    width = qd + 2 * kd + 16
    base, _ = typed(rows_of(5, n, width), bf16)
    starts = [4, 37, 37, 80]
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=-0.11, window=30, causal=False)
    q, k, v = (np.ascontiguousarray(base[:, a:a + d]) for a, d in ((8, qd), (8 + qd, kd), (8 + qd + kd, kd)))
    d = hip_rt.malloc(base.nbytes)
    try:
        with nh.KVCache([32], [32]) as kv:
            plain = kv.attend_packed(q, k, v, starts=starts, **shape)
            hip_rt.to_device(d, base)
            at = [d + size * x for x in (8, 8 + qd, 8 + qd + kd)]
            kv.attend_packed_device(*at, at[0], starts=starts, bf16=bf16, q_stride=width, k_stride=width, v_stride=width,
                                    out_stride=width, **shape)
            kv.sync()
            got = hip_rt.to_host(np.empty_like(base), d)
            alone = np.zeros_like(plain)
            for a, b in zip(starts, starts[1:]):
                if b > a:
                    alone[a:b] = kv.attend_packed(q[a:b], k[a:b], v[a:b], starts=[0, b - a], **shape)
        want = base.copy()
        want[4:80, 8:8 + qd] = plain[4:80]
        assert np.array_equal(got, want) and np.array_equal(plain, alone)
        o, bound = expected(as_values(q), as_values(k), as_values(v), starts, bf16, **shape)
        assert (np.abs(as_values(plain) - o) <= bound)[4:80].all()
    finally:
        hip_rt.free(d)


@pytest.mark.gpu
def test_magnitudes_f32():
    """Values whose size changes from step to step by many powers of ten, large and
    tiny ones, and scales of 0."""
    n, n_head, hd = 400, 2, 64
    starts = [0, 300, n]
    with nh.KVCache([32], [32]) as kv:
        for fq, fk, fv in ((1, 1, 1e30), (1, 1, 1e-30), (1e20, 1e-20, 1), (1e-25, 1e3, 1e-3), (1, 0, 0), (0, 1, 1)):
            q, k, v = rows_of(1, n, n_head * hd) * np.float32(fq), rows_of(2, n, hd) * np.float32(fk), rows_of(3, n, hd) * np.float32(fv)
            for scale in (0.125, 0.0):
                shape = dict(n_head=n_head, n_kv=1, head_dim=hd, scale=scale, window=0, causal=True)
                got = kv.attend_packed(q, k, v, starts=starts, **shape)
                want, bound = expected(*(x.astype(np.float64) for x in (q, k, v)), starts, False, **shape)
                assert (np.abs(got - want) <= bound).all(), (fq, fk, fv, scale)
        # V grows by 10^6 every 70 rows, then shrinks
        v = rows_of(3, n, hd) * np.float32(10.0)**np.float32(6 * (np.minimum(np.arange(n), n - np.arange(n)) // 70))[:, None]
        q, k = rows_of(1, n, n_head * hd), rows_of(2, n, hd)
        shape = dict(n_head=n_head, n_kv=1, head_dim=hd, scale=0.125, window=40, causal=True)
        got = kv.attend_packed(q, k, v, starts=starts, **shape)
        for a, b in zip(starts, starts[1:]):
            for t in range(a, b):  # (a bound per row: its own window's largest |V|)
                f = max(a, t - 39)
                o, d, _ = ref.attend(q[t:t + 1], k[f:t + 1], v[f:t + 1], pos0=t - f, n_seq=t - f + 1,
                                     **dict(shape, window=0))
                assert (np.abs(got[t] - o[0]) <= d[0] + 2.0**-20 * np.abs(v[f:t + 1]).max()).all(), t


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (False, 40)])
def test_infinite_and_nan_elements(bf16, causal, window):
    """Rows that do not attend a key with such an element get their clean values,
    rows that attend an infinite V get it in its column alone; a query's reach its
    own head."""
    n_head, n_kv, hd, n = 4, 2, 64, 300
    starts = [0, 180, n]
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=0.125, window=window, causal=causal)
    q, k, v = rows_of(1, n, n_head * hd), rows_of(2, n, n_kv * hd), rows_of(3, n, n_kv * hd)
    key, g = 75, 2
    sees = np.zeros(n, bool)
    for t in range(180):
        a, b = ref.span(causal, window, t, 180)
        sees[t] = a <= key <= b
    with nh.KVCache([32], [32]) as kv:
        run = lambda *x: as_values(kv.attend_packed(*(typed(y, bf16)[0] for y in x), starts=starts, **shape))  # noqa: E731
        want, bound = expected(*(typed(y, bf16)[1] for y in (q, k, v)), starts, bf16, **shape)
        for name, value in (("v", np.inf), ("v", np.nan), ("k", np.nan), ("k", np.inf), ("q", np.nan)):
            x = dict(q=q.copy(), k=k.copy(), v=v.copy())
            x[name][key, 5] = value
            got = run(x["q"], x["k"], x["v"])
            hit = np.zeros(want.shape, bool)
            if name == "q":
                hit[key, :hd] = True
                assert np.isnan(got[key, :hd]).all()
            elif name == "v":
                hit[sees, 5:g * hd:hd] = True  # column 5 of the KV head's two query heads
                assert (np.isnan(got[hit]) if np.isnan(value) else got[hit] == np.inf).all()
            else:
                hit[sees, :g * hd] = True  # (+-inf scores: NaN, or the key left out)
                if np.isnan(value):
                    assert np.isnan(got[hit]).all()
            assert (np.abs(got - want) <= bound)[~hit].all(), (name, value)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
def test_captured(bf16):
    """Captured without a call before (nothing is allocated), replayed with other
    inputs between eager calls; the caller's starts may change after the capture."""
    n_head, n_kv, hd = 8, 2, 128
    starts = (C.c_int32 * 4)(0, 100, 101, 260)
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=0.09)
    sets = [[typed(rows_of(10 * i + s, 260, h * hd), bf16)[0] for s, h in ((1, n_head), (2, n_kv), (3, n_kv))] for i in range(3)]
    dev = [hip_rt.malloc(x.nbytes) for x in (*sets[0], sets[0][0])]
    try:
        with nh.KVCache([32], [32]) as kv, nh.KVCache([32], [32]) as other:
            graph = hip_rt.Graph(kv.stream, lambda: kv.attend_packed_device(*dev, starts=starts, bf16=bf16, **shape))
            starts[1] = 7
            for x in sets:
                for d, a in zip(dev, x):
                    hip_rt.to_device(d, a)
                graph.launch(kv.stream)
                kv.sync()
                got = hip_rt.to_host(np.empty_like(x[0]), dev[3])
                assert np.array_equal(got, other.attend_packed(*x, starts=[0, 100, 101, 260], **shape))
            graph.close()
    finally:
        for d in dev:
            hip_rt.free(d)


def test_refused_without_a_cache():
    lib = nh.load_library()
    s = (C.c_int32 * 2)(0, 1)
    assert lib.nnc_hip_attend_packed_device(None, 1, 16, 64, 16, 64, 16, 64, 16, 64, s, 1, 0, True, 1, 1, 64, 1.0) == \
        nh.NncStatus.INVALID_ARGUMENT


@pytest.mark.gpu
def test_refusals():
    lib = nh.load_library()
    ok = dict(type=1, q=1 << 20, qs=256, k=2 << 20, ks=128, v=3 << 20, vs=128, out=4 << 20, os=256, starts=[0, 0, 0], n=2,
              window=0, causal=True, h=4, kv=2, hd=64, scale=0.1)  # (addresses of no memory: every sequence is empty)
    with nh.KVCache([32], [32]) as kv:
        def call(**change):
            a = dict(ok, **change)
            st = a["starts"]
            arr = None if st is None else (C.c_int32 * len(st))(*st)
            return lib.nnc_hip_attend_packed_device(kv.handle, a["type"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["out"],
                                                    a["os"], arr, a["n"], a["window"], a["causal"], a["h"], a["kv"], a["hd"],
                                                    a["scale"])
        assert call() == nh.NncStatus.OK and call(n=0, starts=None) == nh.NncStatus.OK
        assert call(type=0) == nh.NncStatus.OK
        for bad in (dict(type=2), dict(type=-1), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(n=-1),
                    dict(starts=None), dict(starts=[-1, 0, 0]), dict(starts=[5, 4, 9]), dict(starts=[0, 3, 2]), dict(window=-1),
                    dict(h=5), dict(h=0), dict(kv=0), dict(kv=-2), dict(hd=0), dict(q=(1 << 20) + 8), dict(out=(1 << 20) + 2),
                    dict(qs=248), dict(ks=120), dict(os=260), dict(vs=1 << 23), dict(qs=(1 << 64) - 8), dict(type=0, ks=130)):
            assert call(**bad) == nh.NncStatus.INVALID_ARGUMENT, bad
            assert lib.nnc_hip_last_error()
        for bad in (dict(hd=60, qs=512, ks=512, vs=512, os=512), dict(hd=264, qs=2048, ks=1024, vs=1024, os=2048)):
            assert call(**bad) == nh.NncStatus.UNSUPPORTED_MODEL, bad


@pytest.mark.gpu
def test_prompts_then_decode_over_four_bits():
    """Two requests as a server runs them: their prompts' attention in one packed
    call over the exact rows, those rows into a 4-bit cache each, then tokens of
    both over the caches."""
    n_head, n_kv, hd = 8, 2, 128
    lens, steps = [150, 61], 5
    starts = [0, 150, 211]
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    q, k, v = rows_of(1, 211, n_head * hd), rows_of(2, 211, n_kv * hd), rows_of(3, 211, n_kv * hd)
    caches = [nh.KVCache([256], [n_kv * hd], q4=True) for _ in lens]
    try:
        got = caches[0].attend_packed(q, k, v, starts=starts, **shape)
        want, bound = expected(*(x.astype(np.float64) for x in (q, k, v)), starts, False, window=0, causal=True, **shape)
        assert (np.abs(got - want) <= bound).all()
        for i, kv in enumerate(caches):
            a, b = starts[i], starts[i + 1]
            kv.append_f32(0, 0, k[a:b], v[a:b])
            kk, vv = k[a:b], v[a:b]
            for t in range(steps):
                q1, k1, v1 = (rows_of(100 * i + 10 * t + s, 1, h * hd) for s, h in ((1, n_head), (2, n_kv), (3, n_kv)))
                kv.append_f32(0, lens[i] + t, k1, v1)
                kk, vv = np.concatenate([kk, k1]), np.concatenate([vv, v1])
                out = kv.attend(0, q1, pos0=lens[i] + t, **shape)
                want, bound, _ = ref.attend(q1, ref.values(ref.quantise(kk)), ref.values(ref.quantise(vv)), pos0=lens[i] + t,
                                            n_seq=lens[i] + t + 1, window=0, causal=True, **shape)
                assert (np.abs(out - want) <= bound).all()
    finally:
        for kv in caches:
            kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
def test_long_sequence_of_few_heads(bf16):
    """One whose keys work-groups share, beside short ones: plain, with an infinite
    and a NaN value in the middle of it, and captured before and after the scratch
    for it is there."""
    n_head, n_kv, hd = 2, 1, 64
    starts = [0, 5, 1905, 1905, 1950]
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=0.125, window=0, causal=True)
    (q, q64), (k, k64), (v, v64) = (typed(rows_of(s, 1950, h * hd), bf16) for s, h in ((1, n_head), (2, n_kv), (3, n_kv)))
    want, bound = expected(q64, k64, v64, starts, bf16, **shape)
    dev = [hip_rt.malloc(x.nbytes) for x in (q, k, v, q)]
    try:
        with nh.KVCache([32], [32]) as kv:
            for d, x in zip(dev, (q, k, v)):
                hip_rt.to_device(d, x)

            def call():
                kv.attend_packed_device(*dev, starts=starts, bf16=bf16, **shape)

            def out():
                kv.sync()
                return hip_rt.to_host(np.empty_like(q), dev[3])

            early = hip_rt.Graph(kv.stream, call)
            early.launch(kv.stream)
            assert (np.abs(as_values(out()) - want) <= bound).all()
            call()
            got = out()
            assert (np.abs(as_values(got) - want) <= bound).all()
            late = hip_rt.Graph(kv.stream, call)
            for _ in range(3):
                late.launch(kv.stream)
                assert np.array_equal(out(), got)
                kv.attend_packed(q[:300], k[:300], v[:300], starts=[0, 300], **shape)
            for key, value in ((900, np.inf), (1700, np.nan)):
                x = as_values(v).astype(np.float32)
                x[5 + key, 7] = value
                hip_rt.to_device(dev[2], typed(x, bf16)[0])
                call()
                y = as_values(out())
                hit = np.zeros(want.shape, bool)
                hit[5 + key:1905, 7::hd] = True
                assert (np.isnan(y[hit]) if np.isnan(value) else y[hit] == np.inf).all()
                assert (np.abs(y - want) <= bound)[~hit].all()
            early.close()
            late.close()
    finally:
        for d in dev:
            hip_rt.free(d)


@pytest.mark.gpu
def test_more_refusals():
    """Operands that out may not be, and sequences past a launch (no memory behind the
    addresses: refused before anything is queued)."""
    with nh.KVCache([32], [32]) as kv:
        ok = dict(starts=[0, 0], bf16=True, n_head=4, n_kv=2, head_dim=64, scale=0.1)
        q, k, v = 1 << 20, 2 << 20, 3 << 20
        kv.attend_packed_device(q, k, v, q, **ok)
        kv.attend_packed_device(q, k, k, q, q_stride=1024, out_stride=1024, **ok)
        for out, more in ((k, {}), (v, {}), (q, dict(q_stride=512)), (q, dict(out_stride=264))):
            with pytest.raises(nh.NncError) as e:
                kv.attend_packed_device(q, k, v, out, **{**ok, **more})
            assert e.value.status == nh.NncStatus.INVALID_ARGUMENT
        with pytest.raises(nh.NncError) as e:
            kv.attend_packed_device(q, k, v, 4 << 20, **{**ok, "starts": [0, 1, 1 + 2**26 + 1]})
        assert e.value.status == nh.NncStatus.UNSUPPORTED_MODEL
        x = rows_of(1, 8, 64)
        for starts, short in (([0, 9], 0), ([0, 8], 1), ([0, 8], 2), ([9, 9], 0)):
            a = [x, x, x]
            a[short] = a[short][:7] if starts[1] == 8 else x
            with pytest.raises(ValueError):
                kv.attend_packed(*a, starts=starts, n_head=1, n_kv=1, head_dim=64, scale=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_largest_stride_and_offsets_past_32_bits(bf16, hd):
    """Rows as far apart as the entry point takes, from a row on whose offset passes
    2^32 bytes."""
    n, at, es = 70, 300 if bf16 else 150, 2 if bf16 else 4
    stride = (1 << 23) - 8
    shape = dict(n_head=2, n_kv=1, head_dim=hd, scale=hd**-0.5, window=0, causal=True)
    (q, q64), (k, k64), (v, v64) = (typed(rows_of(s, n, h * hd), bf16) for s, h in ((1, 2), (2, 1), (3, 1)))
    want, bound = expected(q64, k64, v64, [0, n], bf16, **shape)
    assert at * stride * es > 1 << 32
    print(f"largest stride, head_dim {hd}, bf16 {bf16}", flush=True)
    base = hip_rt.malloc((at + n) * stride * es)
    try:
        where = [base, base + 2 * hd * es, base + 3 * hd * es, base + 4 * hd * es]  # q, k, v, out
        for p, x in zip(where, (q, k, v)):
            for i in range(n):
                hip_rt.to_device(p + (at + i) * stride * es, x[i])
        with nh.KVCache([32], [32]) as kv:
            kv.attend_packed_device(*where, starts=[at, at + n], bf16=bf16, q_stride=stride, k_stride=stride, v_stride=stride,
                                    out_stride=stride, **shape)
            kv.sync()
        got = np.stack([hip_rt.to_host(np.empty_like(q[0]), where[3] + (at + i) * stride * es) for i in range(n)])
    finally:
        hip_rt.free(base)
    assert (np.abs(as_values(got) - want) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("n_head,n_kv,hd,window,causal,lens", [
    (2, 1, 64, 0, True, [3000, 4, 2500, 0, 2000, 700]),  # several sequences share their keys in one launch
    (1, 1, 256, 0, False, [1500, 1501]),
    (64, 1, 16, 0, True, [130]),
    (33, 33, 8, 1, True, [70, 1]),
    (3, 1, 128, 1000, False, [40, 900]),
    (4, 2, 248, 3, False, [100] * 3),
    (2, 2, 40, 0, True, [64] * 70),
])
def test_corners(n_head, n_kv, hd, window, causal, lens, bf16):
    print(f"packed corner {n_head}/{n_kv}/{hd} window {window} causal {causal} bf16 {bf16} {len(lens)} sequences", flush=True)
    starts = [0, *np.cumsum(lens).tolist()]
    shape = dict(window=window, causal=causal, n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    (q, q64), (k, k64), (v, v64) = (typed(rows_of(s, starts[-1], h * hd), bf16) for s, h in ((1, n_head), (2, n_kv), (3, n_kv)))
    with nh.KVCache([32], [32]) as kv:
        got = kv.attend_packed(q, k, v, starts=starts, **shape)
    want, bound = expected(q64, k64, v64, starts, bf16, **shape)
    assert (np.abs(as_values(got) - want) <= bound).all()


@pytest.mark.gpu
def test_shared_scratch_in_one_graph():
    """A packed call and a batch over the same 4-bit cache, both sharing keys and so
    the cache's scratch, one after the other in one graph: every replay has the eager
    calls' bits, other calls on the cache in between."""
    n_head, n_kv, hd, n = 2, 1, 128, 2600
    shape = dict(n_head=n_head, n_kv=n_kv, head_dim=hd, scale=hd**-0.5)
    q, k, v = rows_of(1, n, n_head * hd), rows_of(2, n, n_kv * hd), rows_of(3, n, n_kv * hd)
    starts = [0, 2000, n]
    dev = [hip_rt.malloc(x.nbytes) for x in (q, k, v, q, q)]
    try:
        with nh.KVCache([4096], [n_kv * hd], q4=True) as kv:
            for d, x in zip(dev, (q, k, v)):
                hip_rt.to_device(d, x)
            kv.append_f32(0, 0, k, v)

            def both():
                kv.attend_packed_device(*dev[:4], starts=starts, bf16=False, **shape)
                kv.attend_device(0, dev[0], dev[4], n_tok=30, pos0=n - 30, n_seq=n, window=0, causal=True, **shape)

            def outs():
                kv.sync()
                return hip_rt.to_host(np.empty_like(q), dev[3]), hip_rt.to_host(np.empty_like(q[:30]), dev[4])

            both()
            want = outs()
            graph = hip_rt.Graph(kv.stream, both)
            for i in range(4):
                hip_rt.to_device(dev[3], np.zeros_like(q))
                graph.launch(kv.stream)
                for a, b in zip(outs(), want):
                    assert np.array_equal(a, b), i
                kv.attend(0, q[:20 + i], pos0=n - 20 - i, n_seq=n, **shape)
            graph.close()
    finally:
        for d in dev:
            hip_rt.free(d)
