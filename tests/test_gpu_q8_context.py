"""GPU tests of an 8-bit context (cache_type KV_CACHE_Q8): kv_append, kv_attend,
kv_attend_mask, kv_forward, row export and import, and kv_evict, against the
F16 context on the same values and the 64-bit restatement."""
import numpy as np
import pytest
import torch

import kv_b200 as K
import q8_reference as R

pytestmark = pytest.mark.gpu
B = R.BLOCK


def spec(d=128, hq=8, h=2, layers=2, **kw):
    return dict(dict(n_layer=layers, n_head=hq, n_head_kv=h, head_dim=d, n_rot=d, rope_mode=2, rope_base=10000.0, n_ctx=512), **kw)


def inputs(seed, n, hq, h, d):
    g = torch.Generator().manual_seed(seed)
    fused = torch.randn(n, (hq + 2 * h) * d, generator=g).cuda()
    return fused[:, :hq * d], fused[:, hq * d:(hq + h) * d], fused[:, (hq + h) * d:]


def append(ctx, layer, n_past, qkv, norms=(None, None)):
    q, k, v = qkv
    ctx.append(layer, n_past, q.shape[0], q, q.stride(0), k, k.stride(0), v, v.stride(0), *norms)


def q8_context(sp, **kw):
    return K.Context(K.make_config(sp, cache_type=K.KV_CACHE_Q8, **kw))


def quantised(rows_u16):
    """[n][h][d] F16 bits -> the values an 8-bit cache holds, when the rows were stored in one call."""
    x = rows_u16.view(np.float16).astype(np.float64)
    out = np.empty_like(x)
    for h in range(x.shape[1]):
        for b in range(0, x.shape[0], B):
            c, w = R.quantise_block(x[b:b + B, h])
            out[b:b + B, h] = R.row_values(c, np.array([w], np.uint32))
    return out


SPECS = {"plain": spec(), "normal-rope": spec(rope_mode=0, d=64, hq=6, h=3), "qk-norm": spec(qk_norm=1, rms_eps=1e-6),
         "partial-rope": spec(d=96, hq=4, h=4, n_rot=48), "ngpt-256": spec(d=256, hq=8, h=2, qk_norm=2)}


@pytest.mark.parametrize("name", list(SPECS))
def test_rows_are_the_f16_context_s_in_8_bits(name):
    sp = SPECS[name]
    hq, h, d = sp["n_head"], sp["n_head_kv"], sp["head_dim"]
    g = torch.Generator().manual_seed(1)
    qn = torch.rand(hq * d if sp.get("qk_norm") == 2 else d, generator=g).cuda() + 0.5
    norms = {1: (qn, torch.rand(d, generator=g).cuda() + 0.5), 2: (qn, None)}.get(sp.get("qk_norm"), (None, None))
    with q8_context(sp) as a, K.Context(K.make_config(sp)) as b:
        qkv = inputs(3, 70, hq, h, d)
        for ctx in (a, b):
            append(ctx, 1, 0, qkv, norms)
        torch.cuda.synchronize()
        for which in (0, 1):
            want = quantised(b.export_rows(1, which, 0, 70))
            got = a.export_rows(1, which, 0, 70).view(np.float16).astype(np.float64)
            assert np.array_equal(got, want)
        assert a.layer_rows(1) == (70, 512) and a.layer_rows(0) == (0, 512)


def close(got, want):
    """The framework's attention tolerance (two roundings of the weights to F16)."""
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all()
    assert (got - want).abs().max() <= 2e-3 * max(1.0, float(want.abs().max()))
    assert float((got - want).norm() / want.norm()) <= 1e-3


@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("n_past, n_new", [(0, 1), (33, 1), (200, 5), (90, 40), (5, 200)])
@pytest.mark.parametrize("masked", [False, True])
def test_attend_equals_the_f16_context_over_the_same_values(name, n_past, n_new, masked):
    sp = SPECS[name]
    hq, h, d = sp["n_head"], sp["n_head_kv"], sp["head_dim"]
    qn = torch.ones(hq * d if sp.get("qk_norm") == 2 else d, device="cuda")
    norms = {1: (qn, qn[:d]), 2: (qn, None)}.get(sp.get("qk_norm"), (None, None))
    with q8_context(sp) as a, K.Context(K.make_config(sp)) as b:
        if n_past:
            append(a, 0, 0, inputs(1, n_past, hq, h, d), norms)
        new = inputs(2, n_new, hq, h, d)
        append(a, 0, n_past, new, norms)
        append(b, 0, n_past, new, norms)
        for which in (0, 1):
            b.import_rows(0, which, 0, a.export_rows(0, which, 0, n_past + n_new))
        mask = None
        if masked:
            mask = torch.randn(n_new, n_past + n_new + 3, device="cuda")
            mask[torch.rand(mask.shape, device="cuda") < 0.3] = float("-inf")
            mask[:, 0] = 0.0
        outs = []
        for ctx in (a, b):
            out = torch.empty(n_new, hq * d, device="cuda")
            if masked:
                ctx.attend_mask(0, n_past, n_new, mask, out)
            else:
                ctx.attend(0, n_past, n_new, out)
            ctx.status()
            outs.append(out)
        close(*outs)


def test_forward_over_layers_and_replay():
    sp = spec(layers=3)
    hq, h, d = 8, 2, 128
    g = torch.Generator().manual_seed(5)
    with q8_context(sp) as ctx:
        n = 100
        q, k, v = (torch.randn(3, n + 1, w * d, generator=g).cuda() for w in (hq, h, h))
        outs = [torch.zeros(3, n, hq * d, device="cuda"), torch.zeros(3, 1, hq * d, device="cuda")]

        def layers(i):
            a, m = (0, n) if i == 0 else (n, 1)
            for l in range(3):
                append(ctx, l, a, (q[l, a:a + m], k[l, a:a + m], v[l, a:a + m]))
                ctx.attend(l, a, m, outs[i][l])

        layers(0)
        layers(1)
        torch.cuda.synchronize()
        want = outs[1].clone()
        # the same token through kv_forward's layer loop, one layer stride for q, k and v: a fused buffer
        fused = torch.cat([q[:, n], k[:, n], v[:, n]], 1).contiguous()
        ctx.forward(n, 1, fused, 0, fused[:, hq * d:], 0, fused[:, (hq + h) * d:], 0, fused.stride(0), None, None, 0, outs[1],
                    hq * d)
        torch.cuda.synchronize()
        assert torch.equal(outs[1], want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx.forward(n, 1, fused, 0, fused[:, hq * d:], 0, fused[:, (hq + h) * d:], 0, fused.stride(0), None, None, 0,
                        outs[1], hq * d, stream=torch.cuda.current_stream())
        outs[1].zero_()
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[1], want)


def test_import_and_export_round_trip():
    sp = spec(d=64, hq=4, h=2, layers=1)
    rng = np.random.default_rng(1)
    with q8_context(sp) as ctx:
        x = (rng.standard_normal((100, 2, 64)) * 2).astype(np.float16).view(np.uint16)
        for which in (0, 1):
            ctx.import_rows(0, which, 0, x)
            assert np.array_equal(ctx.export_rows(0, which, 0, 100).view(np.float16).astype(np.float64), quantised(x))
        before = [ctx.export_rows(0, w, 0, 100) for w in (0, 1)]
        # what an 8-bit cache exported goes in again unchanged, also in the middle, rows behind it and V untouched
        ctx.import_rows(0, 0, 0, before[0])
        ctx.import_rows(0, 0, 37, before[0][37:50])
        assert all(np.array_equal(ctx.export_rows(0, w, 0, 100), before[w]) for w in (0, 1))
        assert ctx.layer_rows(0) == (100, 512)


def test_a_budget_of_rows_over_a_long_sequence():
    """Positions go on past the rows a layer holds; each layer is evicted whenever it is full."""
    hq, h, d, budget, rows = 6, 2, 64, 40, 96
    sp = spec(d=d, hq=hq, h=h, layers=2, n_rot=0, n_ctx=400)
    rng = np.random.default_rng(4)
    with q8_context(sp, cache_rows=rows, track_weights=True, n_batch_max=48) as ctx:
        assert ctx.layer_rows(0) == (0, 96)
        kept_rows = [[[] for _ in range(h)] for _ in range(2)]   # the reference's K and V values of each layer and head
        weight = [np.zeros((h, 0)) for _ in range(2)]
        n_past = 0
        for step, n in enumerate([48, 30, 1, 1, 1, 1, 1, 20, 1, 1, 33, 17, 40, 1, 1, 1, 48, 25, 1, 30]):
            for layer in range(2):
                used = ctx.layer_rows(layer)[0]
                if used + n > rows:
                    q, k, v = inputs(999, n, hq, h, d)
                    with pytest.raises(K.KvError) as e:
                        append(ctx, layer, n_past, (q, k, v))
                    assert e.value.code == K.KV_E_RANGE
                    kept = torch.empty(h, budget - n % 7, dtype=torch.int32, device="cuda")
                    keep = kept.shape[1]
                    ctx.evict(layer, keep, 16, kept)
                    for i in range(h):
                        idx = kept[i].tolist()
                        assert idx[-16:] == list(range(used - 16, used)) and idx == sorted(set(idx))
                        # the order by the reference's weights, but where two are as near as the tolerance of a weight
                        left = np.setdiff1d(np.arange(used - 16), idx)
                        if len(left):
                            assert weight[layer][i][left].max() <= weight[layer][i][idx[:-16]].min() * (1 + 1e-4) + 1e-7
                        vals = [np.stack(kept_rows[layer][i])[idx][:, w] for w in (0, 1)]
                        for w in (0, 1):
                            for b in range(0, keep, B):
                                c, word = R.quantise_block(vals[w][b:b + B])
                                vals[w][b:b + B] = R.row_values(c, np.array([word], np.uint32))
                        kept_rows[layer][i] = list(np.stack(vals, 1))
                    weight[layer] = np.stack([weight[layer][i][kept[i].cpu().numpy()] for i in range(h)])
                    assert ctx.layer_rows(layer) == (keep, rows)
                    with pytest.raises(K.KvError) as e:
                        ctx.attend(layer, n_past, n, torch.empty(n, hq * d, device="cuda"))
                    assert e.value.code == K.KV_E_STATE
                    used = keep
                qkv = inputs(100 * step + layer, n, hq, h, d)
                append(ctx, layer, n_past, qkv)
                out = torch.empty(n, hq * d, device="cuda")
                ctx.attend(layer, n_past, n, out)
                ctx.status()
                got = [ctx.export_rows(layer, w, 0, used + n).view(np.float16).astype(np.float64) for w in (0, 1)]
                for i in range(h):
                    old = used // B * B   # (rows before the first block of the new ones keep their values)
                    if old:
                        assert np.array_equal(np.stack([g[:old, i] for g in got], 1), np.stack(kept_rows[layer][i][:old]))
                    kept_rows[layer][i] = list(np.stack([g[:, i] for g in got], 1))
                weight[layer] = np.concatenate([weight[layer], np.zeros((h, n))], 1)
                q = qkv[0].half().double().cpu().reshape(n, h, hq // h, d)
                o = out.double().cpu().reshape(n, h, hq // h, d)
                for i in range(h):
                    kk, vv = (torch.from_numpy(g[:, i]) for g in got)
                    want, wt, mag, err, top = R.attend(kk, vv, torch.ones(used + n, dtype=torch.float64), q[:, i], used)
                    assert ((o[:, i] - want).abs() <= mag * 2.0 ** -10 + 1e-6).all()
                    weight[layer][i] += wt.numpy()
            n_past += n
        assert n_past > 2 * rows


def test_rewinding_after_an_eviction():
    hq, h, d = 4, 2, 64
    sp = spec(d=d, hq=hq, h=h, layers=1, n_rot=0, n_ctx=256)
    with q8_context(sp, cache_rows=64, track_weights=True) as ctx:
        out = torch.empty(60, hq * d, device="cuda")
        append(ctx, 0, 0, inputs(1, 60, hq, h, d))
        ctx.attend(0, 0, 60, out)
        ctx.evict(0, 32, 8)
        for n_past, ok in ((60, True), (55, True), (52, True), (51, False), (1, False)):
            if ok:
                append(ctx, 0, n_past, inputs(2, 1, hq, h, d))
                ctx.attend(0, n_past, 1, out)
                assert ctx.layer_rows(0)[0] == n_past - 28 + 1
            else:
                with pytest.raises(K.KvError) as e:
                    append(ctx, 0, n_past, inputs(2, 1, hq, h, d))
                assert e.value.code == K.KV_E_RANGE
        append(ctx, 0, 0, inputs(3, 5, hq, h, d))   # from the start: nothing is gone
        ctx.attend(0, 0, 5, out)
        assert ctx.layer_rows(0) == (5, 64)
        append(ctx, 0, 5, inputs(3, 1, hq, h, d))


def test_rewinding_after_two_evictions():
    """The second one's recent rows reach back behind the first one's: those do not follow one another in position."""
    hq, h, d = 4, 2, 64
    sp = spec(d=d, hq=hq, h=h, layers=1, n_rot=0, n_ctx=256)
    with q8_context(sp, cache_rows=64, track_weights=True) as ctx:
        out = torch.empty(60, hq * d, device="cuda")
        append(ctx, 0, 0, inputs(1, 60, hq, h, d))
        ctx.attend(0, 0, 60, out)
        ctx.evict(0, 32, 8)   # positions 52 to 59 are the last 8 rows
        append(ctx, 0, 60, inputs(2, 2, hq, h, d))
        ctx.attend(0, 60, 2, out)
        ctx.evict(0, 30, 20)
        for n_past in (51, 45, 42):
            with pytest.raises(K.KvError) as e:
                append(ctx, 0, n_past, inputs(3, 1, hq, h, d))
            assert e.value.code == K.KV_E_RANGE
        append(ctx, 0, 52, inputs(3, 1, hq, h, d))
        ctx.attend(0, 52, 1, out)
        assert ctx.layer_rows(0) == (21, 64)


def test_refusals_of_a_context():
    sp = spec(d=64, hq=4, h=2, layers=1, n_rot=0, n_ctx=100)
    with q8_context(sp, track_weights=True) as ctx:
        append(ctx, 0, 0, inputs(1, 40, 4, 2, 64))
        for args, code in (((0, 41, 0), K.KV_E_ARG), ((0, 0, 0), K.KV_E_ARG), ((0, 10, 11), K.KV_E_ARG),
                           ((0, 10, -1), K.KV_E_ARG), ((1, 10, 1), K.KV_E_ARG)):
            with pytest.raises(K.KvError) as e:
                ctx.evict(*args)
            assert e.value.code == code
        with pytest.raises(K.KvError) as e:
            ctx.fill_synthetic(1, 0, 10)
        assert e.value.code == K.KV_E_UNSUPPORTED
        s = torch.cuda.Stream()
        with pytest.raises(K.KvError) as e:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                ctx.evict(0, 10, 1, stream=s)
        assert e.value.code == K.KV_E_STATE
        ctx.evict(0, 10, 1)
        torch.cuda.synchronize()
    with q8_context(sp) as ctx, K.Context(K.make_config(sp)) as f16:
        for c in (ctx, f16):
            with pytest.raises(K.KvError) as e:
                c.evict(0, 1, 0)
            assert e.value.code == K.KV_E_UNSUPPORTED
        with pytest.raises(K.KvError) as e:
            f16.layer_rows(0)
        assert e.value.code == K.KV_E_UNSUPPORTED


def test_auto_sized_context():
    sp = spec(d=64, hq=4, h=2, layers=1, n_ctx=0, n_ctx_train=3000)
    with q8_context(sp) as ctx:
        assert ctx.n_ctx == 3000
        assert ctx.layer_rows(0) == (0, 3008)


def exported(ctx, layer, row0, n):
    return [ctx.export_rows(layer, w, row0, n) for w in (0, 1)]


def random_rows(seed, n, h, d, size=1.0):
    x = np.random.default_rng(seed).standard_normal((n, h, d)) * size
    return x.astype(np.float16).view(np.uint16)


def test_import_after_a_rewind_takes_no_old_row():
    """What a rewind left behind the rows in use, large values and infinities among them, has no part in an import."""
    hq, h, d = 4, 2, 64
    with q8_context(spec(d=d, hq=hq, h=h, layers=1, n_rot=0)) as ctx:
        big = [x.clone() * 1000.0 for x in inputs(1, 40, hq, h, d)]
        big[1][25, 3] = float("inf")
        append(ctx, 0, 0, big)
        append(ctx, 0, 0, inputs(2, 21, hq, h, d))
        v = exported(ctx, 0, 0, 21)[1]
        x = random_rows(3, 21, h, d)
        ctx.import_rows(0, 0, 0, x)
        got = exported(ctx, 0, 0, 21)
        assert np.array_equal(got[0].view(np.float16).astype(np.float64), quantised(x))
        assert np.array_equal(got[1], v) and ctx.layer_rows(0) == (21, 512)
        # rows behind those in use: the other of K and V holds zeros there until it is imported
        y = random_rows(4, 19, h, d)
        ctx.import_rows(0, 1, 21, y)
        got = exported(ctx, 0, 0, 40)
        assert np.array_equal(got[0][:21].view(np.float16).astype(np.float64), quantised(x)) and not got[0][21:].any()
        both = np.concatenate([v, y])
        # (row 21's block was stored twice: V's rows before it were codes already)
        assert np.array_equal(got[1][32:].view(np.float16).astype(np.float64), quantised(both)[32:])
        assert ctx.layer_rows(0) == (40, 512)


def test_import_behind_the_rows_in_use_leaves_zeros_between():
    hq, h, d = 4, 2, 64
    with q8_context(spec(d=d, hq=hq, h=h, layers=1, n_rot=0)) as ctx:
        append(ctx, 0, 0, inputs(1, 200, hq, h, d))
        append(ctx, 0, 0, inputs(2, 37, hq, h, d))
        before = exported(ctx, 0, 0, 37)
        x = random_rows(3, 10, h, d)
        for w in (0, 1):
            ctx.import_rows(0, w, 100, x)
        got = exported(ctx, 0, 0, 110)
        alone = np.zeros((110, h, d), np.uint16)
        alone[100:] = x
        for g, b in zip(got, before):
            assert np.array_equal(g[:37], b) and not g[37:100].any()
            assert np.array_equal(g[96:].view(np.float16).astype(np.float64), quantised(alone)[96:])
        assert ctx.layer_rows(0) == (110, 512)


def test_import_after_an_eviction_takes_no_row_or_weight_of_another_layer():
    hq, h, d = 4, 2, 64
    sp = spec(d=d, hq=hq, h=h, layers=2, n_rot=0, n_ctx=256)
    with q8_context(sp, cache_rows=64, track_weights=True) as ctx:
        out = torch.empty(60, hq * d, device="cuda")
        for layer, size in ((0, 1.0), (1, 100.0)):
            q, k, v = inputs(layer, 60, hq, h, d)
            append(ctx, layer, 0, (q, k * size if layer else k, v * size))
            ctx.attend(layer, 0, 60, out)
        ctx.evict(1, 40, 8)
        ctx.evict(0, 40, 8)            # layer 0 now has the buffers that were layer 1's
        before = exported(ctx, 0, 0, 40)
        for w in (0, 1):
            ctx.import_rows(0, w, 0, before[w])
        assert all(np.array_equal(a, b) for a, b in zip(exported(ctx, 0, 0, 40), before))
        x = random_rows(7, 12, h, d)
        for w in (0, 1):
            ctx.import_rows(0, w, 40, x)
        assert ctx.layer_rows(0) == (52, 64)
        kept = torch.empty(h, 40, dtype=torch.int32, device="cuda")
        ctx.evict(0, 40, 0, kept)      # the imported rows have no weight, all others some
        assert kept.tolist() == [list(range(40))] * h


def test_a_gap_in_the_positions_is_refused():
    """n_past beyond the rows in use: on a fresh context, after a rewind, and after an eviction."""
    hq, h, d = 4, 2, 64
    sp = spec(d=d, hq=hq, h=h, layers=1, n_rot=0, n_ctx=256)
    with q8_context(sp, cache_rows=128, track_weights=True) as ctx:
        out = torch.empty(60, hq * d, device="cuda")

        def refused(n_past, n=1):
            before = ctx.layer_rows(0)
            with pytest.raises(K.KvError) as e:
                append(ctx, 0, n_past, inputs(9, n, hq, h, d))
            assert e.value.code == K.KV_E_RANGE and ctx.layer_rows(0) == before

        refused(1)
        refused(40, 5)
        append(ctx, 0, 0, inputs(1, 60, hq, h, d))
        ctx.attend(0, 0, 60, out)
        refused(61)
        append(ctx, 0, 10, inputs(2, 1, hq, h, d))   # a rewind: rows 11 to 59 are no longer in use
        refused(12)
        refused(60)
        ctx.attend(0, 10, 1, out)                     # (a refused call leaves the one before it as it was)
        append(ctx, 0, 11, inputs(2, 49, hq, h, d))
        ctx.attend(0, 11, 49, out)
        ctx.evict(0, 32, 8)
        refused(61)
        append(ctx, 0, 60, inputs(3, 1, hq, h, d))
        ctx.attend(0, 60, 1, out)
        assert ctx.layer_rows(0) == (33, 128) and torch.isfinite(out).all()


FAILED_APPEND = """
import ctypes, sys
import torch
import kv_b200 as K
sp = dict(n_layer=1, n_head=4, n_head_kv=2, head_dim=64, n_rot=0, n_ctx=256)
ctx = K.Context(K.make_config(sp, cache_type=K.KV_CACHE_Q8, track_weights=True))
x = torch.randn(40, 8 * 64, device="cuda")
def append(n_past, n, s=None):
    ctx.append(0, n_past, n, x, 512, x[:, 256:], 512, x[:, 384:], 512, stream=s)
append(0, 40)
ctx.evict(0, 20, 8)
out = torch.empty(1, 256, device="cuda")
s = torch.cuda.Stream()
torch.cuda.synchronize()
rt = ctypes.CDLL("libcudart.so.12")
# a capture that an unsupported call has ended: the runtime refuses every launch into its stream
assert rt.cudaStreamBeginCapture(ctypes.c_void_p(s.cuda_stream), 0) == 0
assert rt.cudaDeviceSynchronize() != 0
for n_past in (40, 0):
    try:
        append(n_past, 1, s)
        sys.exit("not refused")
    except K.KvError as e:
        assert e.code == K.KV_E_CUDA, e
    assert ctx.layer_rows(0)[0] == 20
    try:
        ctx.attend(0, n_past, 1, out)
        sys.exit("attend after a failed append")
    except K.KvError as e:
        assert e.code == K.KV_E_STATE, e
g = ctypes.c_void_p()
rt.cudaStreamEndCapture(ctypes.c_void_p(s.cuda_stream), ctypes.byref(g))
rt.cudaGetLastError()
append(40, 1, s)
ctx.attend(0, 40, 1, out, stream=s)
s.synchronize()
assert ctx.layer_rows(0)[0] == 21 and torch.isfinite(out).all()
print("fine")
"""


def test_an_append_that_fails_changes_nothing():
    """In a process of its own, whose runtime refuses the launch."""
    import os
    import subprocess
    import sys
    path = os.path.dirname(os.path.dirname(os.path.abspath(K.__file__)))
    r = subprocess.run([sys.executable, "-c", FAILED_APPEND], env=dict(os.environ, PYTHONPATH=path), capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stdout + r.stderr


def test_attend_after_an_import_of_more_rows():
    """kv_attend goes over the rows up to its kv_append's last one, whatever was imported behind them."""
    sp = spec(d=64, hq=4, h=2, layers=1, n_rot=0)
    for n_past, n_new in ((0, 5), (30, 1), (30, 20)):
        outs = []
        with q8_context(sp) as a, K.Context(K.make_config(sp)) as b:
            if n_past:
                append(a, 0, 0, inputs(1, n_past, 4, 2, 64))
            new = inputs(2, n_new, 4, 2, 64)
            append(a, 0, n_past, new)
            append(b, 0, n_past, new)
            for w in (0, 1):
                a.import_rows(0, w, n_past + n_new, random_rows(w, 90, 2, 64, 3.0))
                b.import_rows(0, w, 0, a.export_rows(0, w, 0, n_past + n_new + 90))
            for ctx in (a, b):
                outs.append(torch.empty(n_new, 4 * 64, device="cuda"))
                ctx.attend(0, n_past, n_new, outs[-1])
            close(*outs)


def test_forward_refuses_before_the_first_layer():
    """A layer without room: no layer's rows or weights change, so the call can be made again after kv_evict."""
    hq, h, d = 4, 2, 64
    sp = spec(d=d, hq=hq, h=h, layers=2, n_rot=0, n_ctx=256)
    with q8_context(sp, cache_rows=64, track_weights=True) as ctx:
        out = torch.empty(2, 64, hq * d, device="cuda")
        for layer in (0, 1):
            append(ctx, layer, 0, inputs(layer, 64, hq, h, d))
            ctx.attend(layer, 0, 64, out[layer])
        ctx.evict(0, 48, 8)
        q, k, v = inputs(5, 4, hq, h, d)
        args = (64, 4, q, q.stride(0), k, k.stride(0), v, v.stride(0), 0, None, None, 0, out, out.stride(0))
        with pytest.raises(K.KvError) as e:
            ctx.forward(*args)
        assert e.value.code == K.KV_E_RANGE
        assert ctx.layer_rows(0) == (48, 64) and ctx.layer_rows(1) == (64, 64)
        ctx.evict(1, 48, 8)
        ctx.forward(*args)
        assert ctx.layer_rows(0) == (52, 64) and ctx.layer_rows(1) == (52, 64)


@pytest.mark.parametrize("n_new", [1, 3, 40])
def test_an_f16_and_an_8_bit_context_in_turn_on_one_stream(n_new):
    """Each step's kernels start while the other context's end; the bits are those of each context alone."""
    sp = spec(layers=2, n_ctx=1200)
    hq, h, d = 8, 2, 128
    steps = [(0, 700), (700, 1), (701, n_new), (701 + n_new, 1), (702 + n_new, 30), (732 + n_new, 1)]
    rows = [[inputs(10 * i + l, n, hq, h, d) for l in range(2)] for i, (_, n) in enumerate(steps)]

    def run(contexts):
        outs = [[torch.full((n, hq * d), 7.0, device="cuda") for _, n in steps for _ in range(2)] for _ in contexts]
        torch.cuda.synchronize()
        for i, (n_past, n) in enumerate(steps):
            for l in range(2):
                for ctx, out in zip(contexts, outs):
                    append(ctx, l, n_past, rows[i][l])
                    ctx.attend(l, n_past, n, out[2 * i + l])
        torch.cuda.synchronize()
        return outs

    def contexts():
        return K.Context(K.make_config(sp, n_batch_max=700)), q8_context(sp, n_batch_max=700)

    a, b = contexts()
    with a, b:
        want = run([a]) + run([b])
    for _ in range(3):
        f16, q8 = contexts()
        with f16, q8:
            got = run([f16, q8])
        for x, y in zip(got, want):
            assert all(torch.equal(s, t) for s, t in zip(x, y))


def prompt_context(**kw):
    """More pairs of tiles than CTAs, several query tiles a KV head, weights kept."""
    hq, h, d = 128, 64, 64
    sp = spec(d=d, hq=hq, h=h, layers=1, n_rot=0, n_ctx=512)
    return q8_context(sp, track_weights=True, **kw), inputs(1, 100, hq, h, d), inputs(2, 400, hq, h, d), hq * d


def expires(what, limit_ms=100):
    """A prompt's chunk with an injected failure: its status is a timeout, once, and the next calls are right."""
    ctx, old, new, width = prompt_context()
    twin = prompt_context()[0]
    with ctx, twin:
        for c in (ctx, twin):
            append(c, 0, 0, old)
        append(ctx, 0, 100, new)
        ctx.debug_inject(what, limit_ns=limit_ms * 1_000_000)
        ctx.attend(0, 100, 400, torch.empty(400, width, device="cuda"))
        with pytest.raises(K.KvError) as e:
            ctx.status()
        assert e.value.code == K.KV_E_TIMEOUT
        assert ctx.status() == K.KV_OK
        ctx.debug_inject(0, limit_ns=1_000_000_000)
        outs = []
        for c in (ctx, twin):
            append(c, 0, 100, new)
            outs.append(torch.empty(400, width, device="cuda"))
            c.attend(0, 100, 400, outs[-1])
            assert c.status() == K.KV_OK
        assert torch.equal(*outs)


def test_a_staging_warp_that_gives_up_alone():
    """The other three are not left at a barrier that it does not come to."""
    expires(3)


@pytest.mark.parametrize("what", [1, 2])
def test_a_wait_that_runs_out(what):
    """In the chunk's kernel, and in the pass that sums its weights."""
    expires(what)


def test_injections_that_do_not_exist():
    with q8_context(spec(d=64, hq=4, h=2, layers=1)) as a, K.Context(K.make_config(spec(d=64, hq=4, h=2, layers=1))) as b:
        for ctx, what in ((a, -1), (a, 4), (b, 2), (b, 3)):
            with pytest.raises(K.KvError) as e:
                ctx.debug_inject(what)
            assert e.value.code == K.KV_E_ARG


def test_a_context_s_status_is_its_own():
    """Neither another 8-bit context nor a caller of the operators takes or sees a context's expired wait."""
    (a, old, new, width), b = prompt_context(), prompt_context()[0]
    c = [torch.zeros(2, 64, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
    direct = K.Q8Cache(*c, *[torch.ones(2, 2, device="cuda") for _ in range(2)])
    with a, b:
        for ctx in (a, b):
            append(ctx, 0, 0, old)
            append(ctx, 0, 100, new)
            if ctx is a:
                a.debug_inject(1, limit_ns=100_000_000)
            ctx.attend(0, 100, 400, torch.empty(400, width, device="cuda"))
        assert b.status() == K.KV_OK and direct.status() == K.KV_OK
        assert direct.status(torch.cuda.Stream()) == K.KV_OK
        with pytest.raises(K.KvError) as e:
            a.status()
        assert e.value.code == K.KV_E_TIMEOUT
        assert a.status() == K.KV_OK


def test_a_chunk_whose_wait_ran_out_adds_no_weights():
    """What kv_evict goes by stays as it was before that call."""
    (a, old, new, width), b = prompt_context(), prompt_context()[0]
    out = torch.empty(400, width, device="cuda")
    kept = []
    with a, b:
        for ctx in (a, b):
            append(ctx, 0, 0, old)
            append(ctx, 0, 100, new)
            ctx.attend(0, 100, 400, out)
            append(ctx, 0, 100, inputs(3, 400, 128, 64, 64))   # the same rows again: their weights are 0
            if ctx is a:
                a.debug_inject(1, limit_ns=100_000_000)
                a.attend(0, 100, 400, out)
                with pytest.raises(K.KvError) as e:
                    a.status()
                assert e.value.code == K.KV_E_TIMEOUT
            kept.append(torch.empty(64, 60, dtype=torch.int32, device="cuda"))
            ctx.evict(0, 60, 0, kept[-1])
        torch.cuda.synchronize()
        assert torch.equal(*kept) and int(kept[0].max()) < 100


@pytest.mark.parametrize("n_past, n_new", [(600, 1), (600, 40), (0, 300)])
@pytest.mark.parametrize("shift", [0.0, 8.0])
def test_the_error_that_the_codes_bring(n_past, n_new, shift):
    """Both contexts on the same rows.  A code is off by up to half a scale, evenly: by scale / sqrt(12) in the mean.  With
    queries and values of size 1 that is the error of a score, and so the relative one of a weight, and that of a value:
    sqrt(sk^2 + sv^2) / sqrt(12) of the outputs, over thousands of them; 1.5 times that is allowed (weights are not all
    small, scales differ from block to block)."""
    hq, h, d = 8, 2, 128
    sp = spec(layers=1, n_rot=0, n_ctx=1024)
    with q8_context(sp) as a, K.Context(K.make_config(sp)) as b:
        outs = []
        for ctx in (a, b):
            for at, n, seed in ((0, 200, 1), (200, n_past - 200, 2), (n_past, n_new, 3)) if n_past else ((0, n_new, 3),):
                q, k, v = inputs(seed, n, hq, h, d)
                k = k.clone()
                k.view(n, h, d)[:, :, :4] += shift   # a few channels of K larger than the others
                append(ctx, 0, at, (q, k, v))
            outs.append(torch.empty(n_new, hq * d, device="cuda"))
            ctx.attend(0, n_past, n_new, outs[-1])
        scale = []
        for which in (0, 1):
            x = b.export_rows(0, which, 0, n_past + n_new).view(np.float16).astype(np.float64)
            words = [R.quantise_block(x[i:i + B, j])[1] for i in range(0, len(x), B) for j in range(h)]
            scale.append(np.sqrt(np.mean(4.0 ** R.word_exp(words))))
        got = float((outs[0] - outs[1]).norm() / outs[1].norm())
        assert 1e-3 < got <= 1.5 * np.hypot(*scale) / np.sqrt(12.0), (got, scale)


@pytest.mark.parametrize("n_past, n_new", [(50, 1), (50, 3), (20, 150)])
def test_many_query_heads_a_kv_head(n_past, n_new):
    """A group of 48: a single token goes to the chunk's kernel."""
    sp = spec(d=64, hq=48, h=1, layers=1)
    with q8_context(sp, track_weights=True) as a, K.Context(K.make_config(sp)) as b:
        append(a, 0, 0, inputs(1, n_past, 48, 1, 64))
        outs = []
        for ctx in (a, b):
            append(ctx, 0, n_past, inputs(2, n_new, 48, 1, 64))
        for which in (0, 1):
            b.import_rows(0, which, 0, a.export_rows(0, which, 0, n_past + n_new))
        for ctx in (a, b):
            outs.append(torch.empty(n_new, 48 * 64, device="cuda"))
            ctx.attend(0, n_past, n_new, outs[-1])
            ctx.status()
        close(*outs)


def test_launches_are_counted_one_by_one():
    with q8_context(spec(layers=1), track_weights=True) as a, q8_context(spec(layers=1)) as b:
        out = torch.empty(64, 8 * 128, device="cuda")

        def launches(ctx, fn):
            n = ctx.launch_count()
            fn()
            return ctx.launch_count() - n

        for ctx in (a, b):
            assert launches(ctx, lambda: append(ctx, 0, 0, inputs(1, 64, 8, 2, 128))) == 2   # the append, the store
        # 64 keys are one sub-tile of a KV head, which one CTA takes: the chunk alone; with weights also their pass
        assert launches(a, lambda: a.attend(0, 0, 64, out)) == 2
        assert launches(b, lambda: b.attend(0, 0, 64, out)) == 1
        for ctx in (a, b):
            append(ctx, 0, 64, inputs(2, 64, 8, 2, 128))
        # 128 are two, cut between CTAs: a fold as well
        assert launches(a, lambda: a.attend(0, 64, 64, out)) == 3
        assert launches(b, lambda: b.attend(0, 64, 64, out)) == 2
        for ctx in (a, b):
            append(ctx, 0, 64, inputs(2, 1, 8, 2, 128))
        # a token over 65 keys, a head a CTA: with weights the join's kernel adds them
        assert launches(a, lambda: a.attend(0, 64, 1, out)) == 2
        assert launches(b, lambda: b.attend(0, 64, 1, out)) == 1
        assert launches(a, lambda: a.evict(0, 40, 4)) == 2
        assert a.status() == b.status() == K.KV_OK
