"""CPU tests of the 8-bit cache's entry points: what they refuse (every check
runs before any CUDA call), and the 64-bit restatement the GPU tests use
against itself."""
import ctypes

import numpy as np
import pytest

import kv_b200 as K
import q8_reference as R

P = 1 << 20   # a stand-in for a device pointer: refused calls never touch it


def cache(**kw):
    d = dict(k=P, v=2 * P, k_scale=3 * P, v_scale=4 * P, weight=5 * P, rows=1024, n_head_kv=2, head_dim=64)
    d.update(kw)
    return K.KvQ8Cache(*[d[n] for n, _ in K.KvQ8Cache._fields_])


BAD_CACHES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(k=P + 8), dict(v=P + 1), dict(k_scale=P + 2),
              dict(weight=P + 1), dict(rows=0), dict(rows=-32), dict(rows=1000), dict(rows=1 << 31), dict(n_head_kv=0),
              dict(n_head_kv=1025), dict(head_dim=80), dict(head_dim=0)]


def store(c, row0=0, n=4, k=6 * P, ks=128, v=7 * P, vs=128, t=0):
    return K.lib().kv_q8_store(ctypes.byref(c) if c else None, row0, n, k, ks, v, vs, t, None)


def load(c, row0=0, n=4, k=6 * P, v=7 * P, s=128, t=0):
    return K.lib().kv_q8_load(ctypes.byref(c) if c else None, row0, n, k, v, s, t, None)


def attend(c, hq=4, past=10, n=2, q=6 * P, qs=256, qt=0, m=0, mt=0, ms=0, fl=0, o=7 * P, os=256, ot=0, w=8 * P,
           wb=1 << 40):
    return K.lib().kv_q8_attend(ctypes.byref(c) if c else None, hq, past, n, q, qs, qt, m, mt, ms, fl, o, os, ot, w, wb,
                                None)


def evict(src, dst, n=100, keep=50, recent=10, kept=100 * P):
    return K.lib().kv_q8_evict(ctypes.byref(src) if src else None, n, keep, recent, ctypes.byref(dst) if dst else None,
                               kept, None)


def other(**kw):
    return cache(**dict(dict(k=11 * P, v=12 * P, k_scale=13 * P, v_scale=14 * P, weight=15 * P), **kw))


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda d: "%s=%s" % next(iter(d.items())))
def test_every_call_refuses_a_bad_cache(bad):
    c = cache(**bad)
    assert store(c) == K.KV_E_ARG
    assert load(c) == K.KV_E_ARG
    assert attend(c) == K.KV_E_ARG
    assert K.lib().kv_q8_attend_workspace(ctypes.byref(c), 4, 10, 2) == 0
    assert evict(c, other()) == K.KV_E_ARG
    assert evict(other(), c) == K.KV_E_ARG
    assert K.last_error()


def test_null_cache():
    assert store(None) == load(None) == attend(None) == evict(None, other()) == evict(cache(), None) == K.KV_E_ARG


@pytest.mark.parametrize("kw, rc", [
    (dict(row0=-1), K.KV_E_RANGE), (dict(n=0), K.KV_E_RANGE), (dict(n=-5), K.KV_E_RANGE), (dict(row0=1021), K.KV_E_RANGE),
    (dict(row0=1 << 62), K.KV_E_RANGE), (dict(n=1025), K.KV_E_RANGE), (dict(k=0), K.KV_E_ARG), (dict(v=0), K.KV_E_ARG),
    (dict(k=6 * P + 2), K.KV_E_ARG), (dict(v=7 * P + 1, t=1), K.KV_E_ARG), (dict(ks=127), K.KV_E_ARG),
    (dict(vs=-128), K.KV_E_ARG), (dict(t=2), K.KV_E_ARG)])
def test_store_refusals(kw, rc):
    assert store(cache(), **kw) == rc


@pytest.mark.parametrize("kw, rc", [
    (dict(row0=-1), K.KV_E_RANGE), (dict(n=0), K.KV_E_RANGE), (dict(row0=1000, n=25), K.KV_E_RANGE),
    (dict(k=0, v=0), K.KV_E_ARG), (dict(s=127), K.KV_E_ARG), (dict(t=-1), K.KV_E_ARG), (dict(k=6 * P + 2), K.KV_E_ARG)])
def test_load_refusals(kw, rc):
    assert load(cache(), **kw) == rc


@pytest.mark.parametrize("kw, rc", [
    (dict(hq=3), K.KV_E_ARG), (dict(hq=0), K.KV_E_ARG), (dict(hq=2 * 129), K.KV_E_ARG), (dict(past=-1), K.KV_E_RANGE),
    (dict(n=0), K.KV_E_RANGE), (dict(past=1023), K.KV_E_RANGE), (dict(n=65536), K.KV_E_RANGE), (dict(q=0), K.KV_E_ARG),
    (dict(o=0), K.KV_E_ARG), (dict(w=0), K.KV_E_ARG), (dict(w=8 * P + 128), K.KV_E_ARG), (dict(q=6 * P + 2), K.KV_E_ARG),
    (dict(o=7 * P + 1, ot=1), K.KV_E_ARG), (dict(qs=255), K.KV_E_ARG), (dict(os=0), K.KV_E_ARG), (dict(qt=2), K.KV_E_ARG),
    (dict(ot=2), K.KV_E_ARG), (dict(m=9 * P, ms=11), K.KV_E_ARG), (dict(m=9 * P, ms=12, mt=2), K.KV_E_ARG),
    (dict(m=9 * P + 2, ms=12), K.KV_E_ARG), (dict(fl=2), K.KV_E_ARG), (dict(wb=0), K.KV_E_RANGE)])
def test_attend_refusals(kw, rc):
    assert attend(cache(), **kw) == rc


def test_attend_refuses_a_workspace_that_is_a_byte_short():
    need = K.lib().kv_q8_attend_workspace(ctypes.byref(cache()), 4, 10, 2)
    assert need > 0
    assert attend(cache(), wb=need - 1) == K.KV_E_RANGE
    assert "workspace" in K.last_error()


def test_workspace_grows_with_the_sizes():
    c = cache(rows=1 << 20, n_head_kv=8, head_dim=128)
    ws = lambda past, n: K.lib().kv_q8_attend_workspace(ctypes.byref(c), 32, past, n)  # noqa: E731
    last = 0
    for past in (0, 1, 31, 500, 4096, 5000, 32768, 131072, 500000):
        here = [ws(past, n) for n in (1, 2, 3, 4, 5, 8, 16, 17, 64, 512)]
        assert here == sorted(here) and here[0] >= last, (past, here)
        last = here[0]


@pytest.mark.parametrize("kw, rc", [
    (dict(keep=0), K.KV_E_ARG), (dict(recent=-1), K.KV_E_ARG), (dict(recent=51), K.KV_E_ARG), (dict(keep=101), K.KV_E_ARG),
    (dict(n=1025), K.KV_E_RANGE), (dict(kept=0), K.KV_E_ARG), (dict(kept=100 * P + 2), K.KV_E_ARG),
    (dict(n=0, keep=0, recent=0), K.KV_E_ARG)])
def test_evict_refusals(kw, rc):
    assert evict(cache(), other(), **kw) == rc


def test_evict_refuses_mismatched_small_and_overlapping_caches():
    assert evict(cache(), other(n_head_kv=1)) == K.KV_E_ARG
    assert evict(cache(), other(head_dim=128)) == K.KV_E_ARG
    assert evict(cache(weight=0), other()) == K.KV_E_ARG
    assert evict(cache(), other(rows=32)) == K.KV_E_RANGE
    assert evict(cache(), cache()) == K.KV_E_ARG
    assert evict(cache(), other(k=2 * P + 16)) == K.KV_E_ARG
    assert evict(cache(), other(v_scale=P + 1024)) == K.KV_E_ARG
    assert evict(cache(), other(), kept=5 * P + 8) == K.KV_E_ARG


def test_reference_block_round_trip():
    rng = np.random.default_rng(1)
    for top in (0.0, 2.0 ** -24, 1e-6, 0.3, 126.9, 127.4, 127.5, 128.0, 65504.0):
        x = rng.uniform(-1, 1, (R.BLOCK, 8)) * top
        x[3, 3] = top
        x = x.astype(np.float16).astype(np.float64)
        c, w = R.quantise_block(x)
        y = R.row_values(c, np.array([w], np.uint32))
        e = int(R.word_exp(w))
        assert np.abs(y - x).max() <= 2.0 ** (e - 1) * (1 if e < 9 else 2)
        c2, w2 = R.quantise_block(y)           # what is stored again keeps its codes and scale
        assert (c2 == c).all() and w2 == w


def test_reference_evict_order():
    w = np.array([1.0, np.nan, 5.0, 5.0, 0.0, -0.0, 5.0, 2.0])
    assert R.evict(w, 8, 4, 1) == [1, 2, 3, 7]
    assert R.evict(w, 8, 8, 0) == list(range(8))
    assert R.evict(w, 8, 3, 3) == [5, 6, 7]
    assert R.evict(w, 7, 6, 0) == [0, 1, 2, 3, 4, 6]


def config(**kw):
    c = K.KvConfig()
    K.lib().kv_config_init(ctypes.byref(c))
    for k, v in dict(dict(n_layer=4, n_head=8, n_head_kv=2, head_dim=64, n_rot=64, n_ctx=1000, cache_type=K.KV_CACHE_Q8),
                     **kw).items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw", [dict(cache_type=2), dict(cache_type=-1), dict(n_shards=2), dict(ring_cells=64),
                                dict(cache_rows=-1), dict(cache_rows=100), dict(cache_rows=100, n_ctx=0, track_weights=1),
                                dict(cache_type=0, cache_rows=5), dict(cache_type=0, track_weights=1),
                                dict(n_head=2 * 129)])
def test_configurations_that_are_refused(kw):
    h = ctypes.c_void_p()
    assert K.lib().kv_alloc(ctypes.byref(config(**kw)), ctypes.byref(h)) == K.KV_E_ARG and not h.value


def test_cache_bytes_of_an_8_bit_configuration():
    block = 2 * (2 * 32 * 64 + 8)
    assert K.cache_bytes(config(), 1000) == 4 * 32 * block
    assert K.cache_bytes(config(track_weights=1), 1000) == 4 * 32 * (block + 2 * 32 * 4)
    assert K.cache_bytes(config(track_weights=1, cache_rows=100), 1000) == 4 * 4 * (block + 2 * 32 * 4)
    assert K.cache_bytes(config(), 0) == 0
    f16 = K.cache_bytes(config(cache_type=0), 1024)
    assert 0.5 * f16 < K.cache_bytes(config(), 1024) < 0.51 * f16


def test_auto_n_ctx_of_an_8_bit_configuration():
    # about twice the F16 cache's positions in the same memory
    a, b = (K.auto_n_ctx(config(cache_type=t, n_layer=32, n_head_kv=8, head_dim=128, n_ctx_train=1 << 30), 100 << 30) for t in (0, 1))
    assert 1.9 * a < b <= 2.0 * a


def test_null_contexts():
    L = K.lib()
    assert L.kv_evict(None, 0, 1, 0, None, None) == K.KV_E_ARG
    assert L.kv_layer_rows(None, 0, None, None) == K.KV_E_ARG


# ---- the Python binding -------------------------------------------------------
def test_a_q8cache_refuses_other_tensors():
    torch = pytest.importorskip("torch")

    def make(k=(2, 64, 64), dtype=torch.int8, v=(2, 64, 64), scale=(2, 2), weight=None, t=False):
        x = torch.zeros(k, dtype=dtype)
        return K.Q8Cache(x.transpose(0, 1) if t else x, torch.zeros(v, dtype=torch.int8), torch.zeros(scale), torch.zeros(scale),
                         None if weight is None else torch.zeros(weight))

    for kw in (dict(dtype=torch.uint8), dict(v=(2, 32, 64)), dict(scale=(2, 64)), dict(weight=(2, 2)), dict(t=True),
               dict()):   # (the last: not on a GPU)
        with pytest.raises(ValueError):
            make(**kw)


def test_the_binding_refuses_other_rows():
    """Its C module's checks, with CPU tensors for a cache on "device -1": nothing here reaches the library but calls it refuses."""
    torch = pytest.importorskip("torch")
    try:
        calls = K._calls()
    except ImportError:
        pytest.skip("the binding's C module is not built")
    c = cache()
    ref = ctypes.addressof(c)
    f, half = lambda *s: torch.zeros(s), lambda *s: torch.zeros(s, dtype=torch.float16)
    good = f(3, 128)
    for k, v in ((f(2, 128), good), (good, f(3, 127)), (good, half(3, 128)), (good.double(), good), (f(3, 256)[:, ::2], good),
                 (f(128, 3).t(), good), (f(128), good), (good, torch.tensor(1.0)), (f(3, 128, 2)[..., 0], good)):
        with pytest.raises(ValueError):
            calls.store(ref, -1, 128, 0, 3, k, v, None)
    with pytest.raises(ValueError):
        calls.store(ref, 0, 128, 0, 3, good, good, None)          # another device
    with pytest.raises(AttributeError):
        calls.store(ref, -1, 128, 0, 3, None, good, None)
    with pytest.raises(TypeError):
        calls.store(ref, -1, 128, 0, 3, good)
    assert calls.store(ref, -1, 128, 1022, 3, good, f(3, 2, 64), None) == K.KV_E_RANGE
    for ko, vo in ((good, half(3, 128)), (good, f(3, 200)[:, :128]), (f(4, 128), None)):
        with pytest.raises(ValueError):
            calls.load(ref, -1, 128, 0, 3, ko, vo, None)
    assert calls.load(ref, -1, 128, 0, 3, None, None, None) == K.KV_E_ARG
    assert calls.load(ref, -1, 128, 1 << 62, 3, good, None, None) == K.KV_E_RANGE
    q, out, ws = f(3, 256), half(3, 4, 64), torch.zeros(64, dtype=torch.uint8)

    def attend(q=q, out=out, mask=None, ws=ws, n_head=4, past=10):
        return calls.attend(ref, -1, 64, n_head, past, 3, q, out, mask, False, ws, None)

    for kw in (dict(q=f(3, 255)), dict(out=f(2, 256)), dict(mask=f(3, 12)), dict(mask=f(2, 13)), dict(mask=f(3, 26)[:, ::2]),
               dict(mask=f(13)), dict(mask=f(3, 13).int()), dict(ws=None), dict(ws=torch.zeros(8, 8)[:, ::2]), dict(n_head=6)):
        with pytest.raises(ValueError):
            attend(**kw)
    assert attend(past=1022) == K.KV_E_RANGE
    kept = torch.zeros(2, 5, dtype=torch.int32)
    d = other()
    for x, dev in ((kept.long(), -1), (kept[:, :4], -1), (kept.t().contiguous(), -1), (kept, 0)):
        with pytest.raises(ValueError):
            calls.evict(ref, -1, 2, 100, 5, 1, ctypes.addressof(d), dev, x, None)
    assert calls.evict(ref, -1, 2, 2000, 5, 1, ctypes.addressof(d), -1, kept, None) == K.KV_E_RANGE


# ---- the kernels' launches ------------------------------------------------------
def test_every_kernel_lets_the_next_one_start_after_its_own_wait():
    """A kernel that starts early may rely on every kernel older than the one before it (the decode attention kernel's first
    tile loads do): that holds where each kernel triggers its dependents only once its own wait is over."""
    import glob
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(K.__file__))), "csrc")
    seen = 0
    for path in sorted(glob.glob(os.path.join(csrc, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for kernel in re.split(r"__global__", text)[1:]:
            name = re.search(r"(\w+)\s*\(const \w+", kernel)
            triggers = [m.start() for m in re.finditer(r"pdl_launch_dependents\(\)", kernel)]
            waits = [m.start() for m in re.finditer(r"pdl_wait\(\)", kernel)]
            for i, t in enumerate(triggers):
                # between one trigger and the next (branches of the kernel) there is a wait
                assert any((triggers[i - 1] if i else 0) <= w < t for w in waits), (path, name and name.group(1))
            seen += len(triggers)
    assert seen >= 10


def test_the_8_bit_kernels_load_nothing_as_read_only():
    """A kernel that starts while the one before it ends must not load what that one writes as constant over its own run."""
    import glob
    import os
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(K.__file__))), "csrc")
    files = glob.glob(os.path.join(csrc, "kv_q8*.cu*"))
    assert len(files) >= 6
    for path in files:
        with open(path) as f:
            text = f.read()
        assert "__ldg" not in text and "global.nc" not in text and "__restrict__" not in text, path


@pytest.mark.parametrize("compiler", ["no-such-compiler", "false"])
def test_the_library_builds_without_a_c_compiler_for_the_binding(tmp_path, monkeypatch, capfd, compiler):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(K.__file__))), "build.py")
    spec = importlib.util.spec_from_file_location("a_build", path)
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    monkeypatch.setenv("CC", compiler)
    monkeypatch.setattr(b, "CALLS", str(tmp_path / "calls.so"))
    monkeypatch.setattr(b, "_compile", lambda src, *a: src)
    monkeypatch.setattr(b, "_stale", lambda target, deps: target == b.CALLS)   # (the library is up to date)
    assert b.build() == b.LIB
    assert "Q8Cache" in capfd.readouterr().err and not os.path.exists(b.CALLS)
    with pytest.raises((OSError, RuntimeError)):
        b.build_calls()


def test_cache_bytes_at_the_largest_sizes():
    top = (1 << 64) - 1
    assert K.cache_bytes(config(), (1 << 63) - 1) == top
    assert K.cache_bytes(config(), 1 << 62) == top
    one = K.cache_bytes(config(n_layer=1, n_head_kv=1, n_head=1), 32)
    assert K.cache_bytes(config(n_layer=1, n_head_kv=1, n_head=1), 1 << 50) == one << 45
    assert K.cache_bytes(config(n_layer=1, n_head_kv=1, n_head=1), (1 << 50) + 1) == (one << 45) + one
    small = config(cache_rows=64, track_weights=1)
    assert K.cache_bytes(small, (1 << 63) - 1) == K.cache_bytes(small, 64)


@pytest.mark.parametrize("channels, shift, stated", [(0, 0.0, 0.017), (4, 8.0, 0.038), (2, 30.0, 0.14)])
def test_the_accuracy_that_the_header_states(channels, shift, stated):
    """The outputs' error that codes bring, by the definition alone: near the figures in kv_api.h and the rule beside them.
    (A rule for the mean of thousands of outputs, whose weights are not all small: a quarter of it is allowed.)"""
    got, rule = [], []
    for seed in range(4):
        rng = np.random.default_rng(seed)
        k, v, q = (rng.standard_normal((n, 128)).astype(np.float16).astype(np.float64) for n in (2048, 2048, 64))
        k[:, :channels] += shift

        def held(x):
            out, scale = np.empty_like(x), []
            for b in range(0, len(x), R.BLOCK):
                c, w = R.quantise_block(x[b:b + R.BLOCK])
                out[b:b + R.BLOCK] = R.row_values(c, np.array([w], np.uint32))
                scale.append(2.0 ** int(R.word_exp(w)))
            return out, np.sqrt(np.mean(np.square(scale)))

        def attend(k, v):
            s = q @ k.T / np.sqrt(128.0)
            p = np.exp(s - s.max(1, keepdims=True))
            return p @ v / p.sum(1, keepdims=True)

        (k8, sk), (v8, sv) = held(k), held(v)
        want = attend(k, v)
        got.append(np.linalg.norm(attend(k8, v8) - want) / np.linalg.norm(want))
        rule.append(np.hypot(sk, sv) / np.sqrt(12.0))
    assert abs(np.mean(got) / np.mean(rule) - 1.0) <= 0.25
    assert abs(np.mean(got) / stated - 1.0) <= 0.1


def test_a_context_s_evict_refuses_other_tensors():
    """A tensor in host memory among them, whose address the kernel would write to.  (The checks come before the library's call,
    which refuses the missing context.)"""
    torch = pytest.importorskip("torch")
    ctx = object.__new__(K.Context)
    ctx.h, ctx.n_kv_heads = None, 2
    try:
        for kept in (torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2, 4, dtype=torch.int32),
                     torch.zeros(5, 2, dtype=torch.int32).t()):
            with pytest.raises(ValueError):
                ctx.evict(0, 5, 1, kept)
        with pytest.raises(K.KvError) as e:
            ctx.evict(0, 5, 1)
        assert e.value.code == K.KV_E_ARG
    finally:
        ctx.h = None
