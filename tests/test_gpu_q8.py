"""GPU tests of the 8-bit cache (kv_q8_store / _load / _attend / _evict) against
their definition in 64 bits (tests/q8_reference.py).  Codes, scales, kept rows
and loaded values are compared bit for bit; attention within the tolerances
that `check` derives."""
import numpy as np
import pytest
import torch

import kv_b200 as K
import q8_reference as R

pytestmark = pytest.mark.gpu
B = R.BLOCK


def rows_of(rng, n, h, d, spread=0.0):
    """Rows with a few large channels; spread: rows' sizes over 2^+-spread."""
    x = rng.standard_normal((n, h, d)) * (0.5 + 2.0 * rng.random((1, h, d)) ** 6)
    return (x * 2.0 ** rng.uniform(-spread, spread, (n, h, 1))).astype(np.float32)


class Cache:
    """A Q8Cache and the reference's copy of it."""

    def __init__(self, h, rows, d, weight=False, seed=0):
        rng = np.random.default_rng(seed)
        # what no row was stored in holds rubbish: codes of every kind, scales that are zeros, NaN, inf or no powers of two
        self.codes = [rng.integers(-128, 128, (h, rows, d)).astype(np.int8) for _ in range(2)]
        rubbish = np.array([0, 0x7FC00000 | 127, 0x7F800000, 0xFF800000, 0x80000000, 0x7FFFFFFF, 0x00000001, 0x7F7FFFFF, 0xC1234567],
                           np.uint32)
        self.words = [rubbish[rng.integers(0, len(rubbish), (h, rows // B))] for _ in range(2)]
        for w in self.words:
            w[:, 0] = 0x7FC00000 | 127
        dev = [torch.from_numpy(c).cuda() for c in self.codes]
        dev += [torch.from_numpy(w.view(np.float32)).cuda() for w in self.words]
        self.w = torch.zeros(h, rows, device="cuda") if weight else None
        self.dev = dev
        self.h, self.rows, self.d = h, rows, d
        self.q8 = K.Q8Cache(*dev, self.w)

    def store(self, row0, k, v, f16=False, device=True):
        """k, v [n][h][d] float32."""
        if device:
            t = torch.float16 if f16 else torch.float32
            kk, vv = (torch.from_numpy(x).cuda().to(t) for x in (k, v))
            self.q8.store(row0, k.shape[0], kk, vv)
        for c, w, x in zip(self.codes, self.words, (k, v)):
            R.store(c, w, row0, x)

    def check(self, n):
        """The first n rows' codes and their blocks' scales, bit for bit; rows behind n as they were."""
        for c, w, dc, dw in zip(self.codes, self.words, self.dev[:2], self.dev[2:]):
            assert np.array_equal(dc.cpu().numpy(), c)
            assert np.array_equal(dw.cpu().numpy().view(np.uint32)[:, :-(-n // B)], w[:, :-(-n // B)])

    def values(self, n, h, attended=False):
        """K and V of head h; attended: as attention sees them, every row of a block with a NaN scale a NaN."""
        got = []
        for c, w in zip(self.codes, self.words):
            x = R.row_values(c[h, :n], w[h])
            if attended:
                x[np.repeat(np.isnan(w[h].view(np.float32)), B)[:n]] = np.nan
            got.append(torch.from_numpy(x))
        return got


def filled(h, n, d, weight=False, seed=0, spread=0.0, extra=B):
    c = Cache(h, -(-n // B) * B + extra, d, weight, seed)
    rng = np.random.default_rng(seed + 1)
    c.store(0, rows_of(rng, n, h, d, spread), rows_of(rng, n, h, d, spread))
    return c


# ---- store and load ----------------------------------------------------------
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("f16", [False, True])
def test_store_in_pieces_matches_the_definition(d, f16):
    rng = np.random.default_rng(d)
    c = Cache(3, 160, d)
    at = 0
    for n in (1, 1, 5, 24, 1, 1, 31, 2, 33, 40):
        c.store(at, rows_of(rng, n, 3, d, 3.0), rows_of(rng, n, 3, d, 3.0), f16)
        at += n
        c.check(at)


@pytest.mark.parametrize("size", [0.0, 1e-7, 6e-8, 1e-3, 127.4, 127.5, 60000.0, 65500.0])
def test_store_at_every_scale(size):
    rng = np.random.default_rng(3)
    c = Cache(2, 64, 64)
    x = rng.uniform(-1, 1, (40, 2, 64)).astype(np.float32) * np.float32(size)
    x[7] = np.float32(size)
    c.store(0, x, -x)
    c.check(40)


def test_store_again_over_rewound_rows():
    rng = np.random.default_rng(5)
    c = Cache(2, 128, 128)
    big = rows_of(rng, 50, 2, 128) * 100
    c.store(0, rows_of(rng, 20, 2, 128), rows_of(rng, 20, 2, 128))
    c.store(20, big, big)          # grows block 0's scale
    c.store(20, rows_of(rng, 3, 2, 128), rows_of(rng, 3, 2, 128))   # and the rows that grew it are gone
    c.check(23)
    c.store(0, big[:1], big[:1])   # from the start
    c.check(1)


def test_store_of_values_that_are_not_finite_and_their_rewind():
    rng = np.random.default_rng(6)
    c = Cache(2, 64, 64)
    x = rows_of(rng, 40, 2, 64)
    c.store(0, x[:10], x[:10])
    y = x[10:20].copy()
    y[3, 0, 5] = np.inf
    y[4, 1, 0] = np.nan
    y[5, 1, 63] = -70000.0         # an F16 infinity
    c.store(10, y, y)
    c.check(20)
    k = torch.empty(20, 2, 64, device="cuda")
    c.q8.load(0, 20, k, None)
    want = np.stack([c.values(20, h)[0].numpy() for h in range(2)], 1)
    assert np.array_equal(k.cpu().numpy(), want.astype(np.float32), equal_nan=True)
    c.store(20, x[20:21], x[20:21])   # the codes survive another store into the block
    c.check(21)
    c.store(10, x[10:40], x[10:40])   # the rows are rewound: their block is finite again
    c.check(40)
    assert not np.isnan(c.dev[2].cpu().numpy()[:, :2]).any()


@pytest.mark.parametrize("f16, pad, shift", [(False, 0, 0), (False, 4, 0), (False, 3, 1), (True, 8, 0), (True, 5, 1)])
def test_strided_and_unaligned_rows(f16, pad, shift):
    h, d, n = 4, 96, 37
    t = torch.float16 if f16 else torch.float32
    wide = torch.randn(n, 2 * h * d + pad + shift, device="cuda").to(t)
    k, v = wide[:, shift:shift + h * d], wide[:, shift + h * d:shift + 2 * h * d]
    c = Cache(h, 64, d)
    c.q8.store(5, n, k, v)
    a, b = (x.float().cpu().numpy().reshape(n, h, d) for x in (k, v))
    # rows 0-4 of the first block hold the rubbish they were made with (at a NaN scale of exponent 0)
    c.store(5, a, b, device=False)
    c.check(42)
    out = torch.zeros_like(wide)
    c.q8.load(5, n, out[:, shift:shift + h * d], out[:, shift + h * d:shift + 2 * h * d])
    for x, cc, ww in ((out[:, shift:shift + h * d], c.codes[0], c.words[0]),
                      (out[:, shift + h * d:shift + 2 * h * d], c.codes[1], c.words[1])):
        want = np.stack([R.row_values(cc[i], ww[i])[5:42] for i in range(h)], 1).reshape(n, h * d)
        assert np.array_equal(x.float().cpu().numpy(), want, equal_nan=True)
    assert not out[:, shift + 2 * h * d:].any() and not out[:, :shift].any()


def test_store_clears_the_new_rows_weights_only():
    c = filled(2, 40, 64, weight=True)
    c.w.fill_(3.0)
    x = np.ones((5, 2, 64), np.float32)
    c.store(33, x, x)
    want = torch.full((2, c.rows), 3.0)
    want[:, 33:38] = 0.0
    assert torch.equal(c.w.cpu(), want)


# ---- attend ------------------------------------------------------------------
def check(c, hq, n_past, n_new, q, mask=None, flash=False, out_f16=False, w0=None, out=None, workspace=None):
    """Runs attend and compares.  Tolerance of an output: a weight's relative error is at most twice the error of a
    score (its own and the sum's), 2^-21 for the exponential, n 2^-24 for the sum of n weights, and half a step of F16
    (2^-11) where the weights are rounded to it: of itself, or 2^-25 below F16's normal numbers, where the largest weight
    times scale is held at 2^7 or more, so 2^-32 of that a key of at most 127; an F16 output adds half a step of itself."""
    n_kv, r, d = n_past + n_new, hq // c.h, c.d
    if out is None:
        out = torch.full((n_new, hq * d), 7.0, device="cuda", dtype=torch.float16 if out_f16 else torch.float32)
    if workspace is None:
        workspace = torch.randint(0, 256, (c.q8.attend_workspace(hq, n_past, n_new),), dtype=torch.uint8, device="cuda")
    c.q8.attend(hq, n_past, n_new, q, out, mask=mask, flash=flash, workspace=workspace)
    got = out.float().cpu().double().view(n_new, c.h, r, d)
    qq = q.half().double().cpu().reshape(n_new, c.h, r, d)
    m = None if mask is None else mask.float().cpu()
    for h in range(c.h):
        k, v = c.values(n_kv, h, True)
        vs = torch.from_numpy(2.0 ** R.word_exp(np.repeat(c.words[1][h], B)[:n_kv]))
        want, weight, mag, err, top = R.attend(k, v, vs, qq[:, h], n_past, m, flash)
        rel = (2 * err + 2.0 ** -21 + n_kv * 2.0 ** -24)[..., None]
        tol = mag * (rel + 2.0 ** -11) + (n_kv * 127 * 2.0 ** -32 * top)[..., None] + 2.0 ** -24
        if out_f16:
            tol = tol + want.abs().nan_to_num() * 2.0 ** -11 + 2.0 ** -25
        assert torch.equal(torch.isnan(got[:, h]), torch.isnan(want)), "NaN rows of head %d" % h
        far = (got[:, h] - want).abs() - tol
        assert not (far > 0).any(), "head %d: over the tolerance by %g" % (h, far[~torch.isnan(far)].max())
        if c.w is not None:
            w = c.w[h].cpu().double()
            old = torch.zeros(c.rows, dtype=torch.float64) if w0 is None else w0[h].double()
            most = weight * (2 * err.max() + 2.0 ** -21 + n_kv * 2.0 ** -24) + \
                (old[:n_kv].abs() + weight) * (n_new * r + 1) * 2.0 ** -24 + 1e-30
            assert not ((w[:n_kv] - old[:n_kv] - weight).abs() > most).any(), "weights of head %d" % h
            assert torch.equal(w[n_kv:], old[n_kv:])
    return out


def queries(seed, n_new, hq, d, f16=True, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n_new, hq * d, generator=g) * size).to(torch.float16 if f16 else torch.float32).cuda()


# query rows a KV head: 1, 2, 7, 8 | 9, 16 | 17, 32 | 33, 64 | 65 and more
SHAPES = [(1, 1, 1), (2, 2, 1), (2, 14, 1), (4, 32, 1), (3, 3, 9), (2, 8, 4), (2, 10, 4), (1, 8, 4), (2, 6, 11), (1, 4, 16),
          (2, 10, 13), (1, 7, 19), (2, 8, 40), (1, 16, 17)]


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("h, hq, n_new", SHAPES)
@pytest.mark.parametrize("n_past", [0, 1, 30, 97, 700])
def test_attend_causal(d, h, hq, n_new, n_past):
    c = filled(h, n_past + n_new, d, weight=True, seed=n_past)
    check(c, hq, n_past, n_new, queries(n_past, n_new, hq, d))


@pytest.mark.parametrize("d, h, hq, n_past, n_new", [(128, 2, 8, 9000, 1), (64, 1, 7, 20011, 1), (96, 2, 2, 5000, 6),
                                                     (256, 1, 4, 4100, 3), (128, 1, 4, 6000, 40), (64, 2, 4, 3000, 300),
                                                     (128, 8, 32, 2500, 1), (128, 1, 8, 2049, 129), (64, 8, 8, 2600, 33),
                                                     (96, 8, 24, 2450, 70), (128, 8, 32, 2500, 40), (128, 16, 16, 1300, 600)])
@pytest.mark.parametrize("weight", [False, True])
def test_attend_long(d, h, hq, n_past, n_new, weight):
    c = filled(h, n_past + n_new, d, weight=weight, seed=1)
    if weight:
        c.w.uniform_(0.0, 2.0)
    w0 = c.w.cpu().clone() if weight else None
    check(c, hq, n_past, n_new, queries(2, n_new, hq, d, f16=False, size=2.0), w0=w0, out_f16=not weight)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("flash", [False, True])
@pytest.mark.parametrize("h, hq, n_new, n_past", [(2, 8, 1, 333), (2, 8, 3, 333), (1, 5, 9, 333), (2, 12, 30, 333),
                                                  (10, 20, 21, 2000)])
def test_attend_mask(f16, flash, h, hq, n_new, n_past):
    d = 128
    n_kv = n_past + n_new
    c = filled(h, n_kv, d, weight=True)
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(n_new, n_kv + 7, generator=g)
    wide[torch.rand(wide.shape, generator=g) < 0.3] = float("-inf")
    wide[:, 64:200] = float("-inf")        # whole tiles removed
    if n_new > 1:
        wide[1] = float("-inf")            # a row with no key
        wide[2, 5:] = float("-inf")        # and one with few
        wide[2, 3] = 0.0
    mask = wide.to(torch.float16 if f16 else torch.float32).cuda()
    check(c, hq, n_past, n_new, queries(9, n_new, hq, d), mask=mask, flash=flash)
    check_again = mask[:, 1:n_kv + 1] if n_new > 1 else mask[:, :n_kv]   # rows off every boundary
    c.w.zero_()
    check(c, hq, n_past, n_new, queries(9, n_new, hq, d), mask=check_again, flash=flash)


@pytest.mark.parametrize("low", [-3.4028234663852886e38, -65504.0])
@pytest.mark.parametrize("n_new", [1, 20])
def test_mask_of_the_lowest_value(low, n_new):
    """Keys masked with the type's lowest value instead of -inf: negligible beside others, equal among themselves."""
    h, hq, d, n_past = 2, 8, 64, 150
    n_kv = n_past + n_new
    c = filled(h, n_kv, d, weight=True, spread=4.0)
    mask = torch.zeros(n_new, n_kv)
    mask[:, ::3] = low
    if n_new > 1:
        mask[3] = low
    if n_new == 1 and low < -1e30:
        mask[:] = low
    check(c, hq, n_past, n_new, queries(1, n_new, hq, d), mask=mask.cuda())


@pytest.mark.parametrize("n_new", [1, 12, 40])
def test_scales_far_apart(n_new):
    """Blocks whose scales differ by up to 2^30, in K and V."""
    h, hq, d, n = 1, 8, 128, 512
    rng = np.random.default_rng(8)
    c = Cache(h, n + n_new + B - (n + n_new) % B, d, True)
    size = np.repeat(2.0 ** rng.integers(-20, 10, n // B + 8), B)[:n + n_new, None, None]
    k = rows_of(rng, n + n_new, h, d)
    v = (rows_of(rng, n + n_new, h, d) * size).astype(np.float32)
    k[64:96] *= 200.0
    k[128:160] *= 1e-6
    c.store(0, k, v)
    check(c, hq, n, n_new, queries(3, n_new, hq, d, size=0.5))


@pytest.mark.parametrize("n_new", [1, 5, 33])
def test_rows_that_are_not_finite(n_new):
    """NaN blocks make the rows that see one of their keys NaN, and only those; masked keys do not enter."""
    h, hq, d, n_past = 2, 6, 96, 200
    n_kv = n_past + n_new
    rng = np.random.default_rng(2)
    c = Cache(h, 256, d, True)
    k, v = rows_of(rng, n_kv, h, d), rows_of(rng, n_kv, h, d)
    k[70, 0, 3] = np.nan      # block 2 of head 0
    v[130, 1, 9] = np.inf     # block 4 of head 1
    c.store(0, k, v)
    mask = torch.zeros(n_new, n_kv)
    mask[:, 64:96] = float("-inf")
    mask[:, 128:160] = float("-inf")
    check(c, hq, n_past, n_new, queries(1, n_new, hq, d), mask=mask.cuda())
    c.w.zero_()
    check(c, hq, n_past, n_new, queries(1, n_new, hq, d))
    mask[:, 66] = 0.0
    c.w.zero_()
    check(c, hq, n_past, n_new, queries(1, n_new, hq, d), mask=mask.cuda())


def test_queries_that_are_not_finite():
    c = filled(2, 100, 64, weight=True)
    q = queries(1, 3, 4, 64)
    q[1, 70] = float("nan")
    q[2, 200] = float("inf")
    out = torch.zeros(3, 4 * 64, device="cuda")
    ws = torch.empty(c.q8.attend_workspace(4, 97, 3), dtype=torch.uint8, device="cuda")
    c.q8.attend(4, 97, 3, q, out, workspace=ws)
    bad = torch.isnan(out).view(3, 4, 64).all(-1).cpu()
    assert bad.tolist() == [[False] * 4, [False, True, False, False], [False, False, False, True]]
    assert torch.isfinite(c.w).all() and abs(float(c.w.sum()) - 10.0) < 1e-4


@pytest.mark.parametrize("pad, shift", [(0, 0), (8, 0), (5, 1)])
def test_strided_queries_and_outputs(pad, shift):
    h, hq, d, n_past, n_new = 2, 6, 64, 75, 7
    c = filled(h, n_past + n_new, d)
    wide = queries(5, n_new, hq, d).new_zeros(n_new, hq * d + pad + shift)
    wide[:, shift:shift + hq * d] = queries(5, n_new, hq, d)
    q = wide[:, shift:shift + hq * d]
    got = torch.full((n_new, hq * d + pad + shift), 9.0, device="cuda")
    check(c, hq, n_past, n_new, q, out=got[:, shift:shift + hq * d])
    assert (got[:, :shift] == 9.0).all() and (got[:, shift + hq * d:] == 9.0).all()


# enough blocks a CTA that the few-row kernel takes its wider form: heads that lie in one CTA, and heads cut between CTAs
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d, h, r, n_past, n_new", [(64, 148, 1, 930, 1), (128, 148, 2, 900, 3), (96, 150, 1, 990, 4),
                                                    (128, 6, 4, 22300, 1), (64, 7, 7, 20000, 1), (96, 5, 2, 28700, 2)])
def test_attend_many_blocks(d, h, r, n_past, n_new, masked):
    n_kv, weight = n_past + n_new, h == 6
    c = filled(h, n_kv, d, weight=weight, seed=3)
    mask = None
    if masked:
        mask = torch.randn(n_new, n_kv, generator=torch.Generator().manual_seed(5))
        mask[:, 40:n_kv // 2] = float("-inf")
        if n_new > 1:
            mask[0] = float("-inf")
        mask = mask.half().cuda()
    check(c, h * r, n_past, n_new, queries(8, n_new, h * r, d), mask=mask, flash=True)


def test_two_streams_at_once():
    """Calls on two streams, each with its workspace, give the bits of the same calls one after the other."""
    c = filled(8, 6000, 128)
    calls = [(1, 5999), (4, 5000), (40, 3000), (100, 5900)]
    qs = [queries(i, n, 32, 128) for i, (n, _) in enumerate(calls)]
    wss = [torch.empty(max(c.q8.attend_workspace(32, p, n) for n, p in calls), dtype=torch.uint8, device="cuda") for _ in range(2)]
    want = []
    for q, (n, past) in zip(qs, calls):
        want.append(torch.empty(n, 32 * 128, device="cuda"))
        c.q8.attend(32, past, n, q, want[-1], workspace=wss[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.full_like(w, 9.0) for w in want] for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(len(calls)):
            for j, st in enumerate(streams):   # (the second stream takes them in the other order)
                m = len(calls) - 1 - i if j else i
                c.q8.attend(32, calls[m][1], calls[m][0], qs[m], outs[j][m], workspace=wss[j], stream=st)
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, w) for x, w in zip(o, want))


@pytest.mark.parametrize("n_new", [1, 3, 9, 40])
def test_offsets_that_pass_32_bits(n_new):
    """A cache of 6.4 GB each of K and V: rows at both ends of every head, the keys between them masked."""
    h, d, rows = 3, 256, 8400000 // B * B
    n_past = rows - n_new - 5
    n_kv = n_past + n_new
    g = torch.Generator(device="cuda").manual_seed(2)
    codes = [torch.empty(h, rows, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    for x in codes:
        for i in range(h):   # (zeros but for the two ends; no row is read that is not one of these)
            x[i].zero_()
            x[i, :64] = torch.randint(-127, 128, (64, d), generator=g, device="cuda", dtype=torch.int8)
            x[i, -96:] = torch.randint(-127, 128, (96, d), generator=g, device="cuda", dtype=torch.int8)
    scales = [torch.full((h, rows // B), 2.0 ** -6, device="cuda") for _ in range(2)]
    q8 = K.Q8Cache(*codes, *scales)
    seen = torch.cat([torch.arange(60), torch.arange(n_kv - 70, n_kv)])
    mask = torch.full((n_new, n_kv), float("-inf"), dtype=torch.float16, device="cuda")
    mask[:, seen.cuda()] = torch.randn(n_new, len(seen), generator=g, device="cuda").half()
    q = queries(4, n_new, h, d)
    out = torch.empty(n_new, h * d, device="cuda")
    ws = torch.empty(q8.attend_workspace(h, n_past, n_new), dtype=torch.uint8, device="cuda")
    q8.attend(h, n_past, n_new, q, out, mask=mask, workspace=ws)
    back = [torch.empty(70, h, d, device="cuda") for _ in range(2)]
    q8.load(n_kv - 70, 70, *back)
    qq, m = q.double().cpu().view(n_new, h, 1, d), mask[:, seen.cuda()].float().cpu()
    for i in range(h):
        k, v = (torch.cat([x[i, :60], x[i, n_kv - 70:n_kv]]).double().cpu() * 2.0 ** -6 for x in codes)
        want, _, mag, err, _ = R.attend(k, v, torch.ones(len(seen), dtype=torch.float64), qq[:, i], 0, m)
        # (the tolerance of `check`, for the keys that are seen)
        tol = mag * ((2 * err + 2.0 ** -21 + len(seen) * 2.0 ** -24)[..., None] + 2.0 ** -11) + 130 * 127 * 2.0 ** -38 + 2.0 ** -24
        assert ((out.double().cpu().view(n_new, h, 1, d)[:, i] - want).abs() <= tol).all()
        for x, y in zip(back, (k, v)):
            assert torch.equal(x[:, i].double().cpu(), y[60:])


def test_the_same_call_gives_the_same_bits():
    c = filled(4, 5000, 128, weight=True)
    q = queries(1, 2, 16, 128)
    ws = torch.empty(c.q8.attend_workspace(16, 4990, 2), dtype=torch.uint8, device="cuda")
    outs = []
    for _ in range(5):
        c.w.zero_()
        out = torch.empty(2, 16 * 128, device="cuda")
        c.q8.attend(16, 4990, 2, q, out, workspace=ws)
        outs.append((out, c.w.clone()))
    assert all(torch.equal(o, outs[0][0]) and torch.equal(w, outs[0][1]) for o, w in outs)


# ---- evict -------------------------------------------------------------------
def run_evict(c, n, keep, recent, with_weight=True, seed=1):
    d = Cache(c.h, -(-keep // B) * B + B, c.d, with_weight, seed=99)
    if with_weight:
        d.w.fill_(-1.0)
    kept = torch.full((c.h, keep), -1, dtype=torch.int32, device="cuda")
    c.q8.evict(n, keep, recent, d.q8, kept)
    w = c.w.cpu().numpy()
    for h in range(c.h):
        want = R.evict(w[h], n, keep, recent)
        assert kept[h].tolist() == want
        for codes, words, cc, ww in zip(c.codes, c.words, d.codes, d.words):
            x = R.row_values(codes[h], words[h])[want]
            for b in range(-(-keep // B)):
                lo, hi = b * B, min(keep, b * B + B)
                cc[h, lo:hi], ww[h, b] = R.quantise_block(x[lo:hi])
        if with_weight:
            got = d.w[h].cpu().numpy()
            assert np.array_equal(got[:keep], w[h][want], equal_nan=True) and (got[keep:] == -1.0).all()
    d.check(keep)
    return d


@pytest.mark.parametrize("h, d, n, keep, recent", [
    (2, 64, 2047, 1023, 127), (1, 128, 33, 1, 0), (1, 128, 33, 1, 1), (3, 96, 100, 100, 3), (3, 96, 100, 99, 0),
    (2, 256, 500, 77, 76), (8, 128, 4001, 1500, 300), (1, 64, 40000, 12345, 678), (2, 64, 1, 1, 0), (5, 128, 1025, 1024, 1024)])
def test_evict(h, d, n, keep, recent):
    c = filled(h, n, d, weight=True, spread=3.0)
    c.w.copy_(torch.randn(c.w.shape, generator=torch.Generator().manual_seed(n)).exp())
    run_evict(c, n, keep, recent)


def test_evict_more_candidates_than_shared_memory_holds():
    n, keep, recent, d = 8 * 32768 + 5001, 70001, 1001, 64
    c = Cache(1, -(-n // B) * B, d, weight=True)
    for w, dw in zip(c.words, c.dev[2:]):
        w[:] = 127 - 6 << 23
        dw.copy_(torch.from_numpy(w.view(np.float32)))
    c.w.copy_(torch.randint(0, 60000, c.w.shape, generator=torch.Generator().manual_seed(1)).float())   # (with ties)
    run_evict(c, n, keep, recent)


@pytest.mark.parametrize("kind", ["zeros", "ties", "nan", "signs", "one", "inf"])
def test_evict_orders_every_weight(kind):
    n = 3000
    c = filled(2, n, 64, weight=True)
    g = torch.Generator().manual_seed(7)
    w = torch.randint(0, 5, c.w.shape, generator=g).float()
    if kind == "zeros":
        w.zero_()
    elif kind == "nan":
        w[:, ::17] = float("nan")
    elif kind == "signs":
        w = torch.randn(c.w.shape, generator=g)
        w[:, ::5] = -0.0
        w[:, 1::5] = 0.0
    elif kind == "one":
        w.zero_()
        w[:, 1234] = 1e-38
        w[:, 99] = 1e-44      # (below the smallest normal number)
    elif kind == "inf":
        w[:, ::900] = float("inf")
    c.w.copy_(w)
    run_evict(c, n, 1000, 100)


def test_evict_into_a_cache_without_weights():
    c = filled(2, 200, 64, weight=True)
    c.w.uniform_()
    run_evict(c, 200, 50, 10, with_weight=False)


def test_evict_moves_values_that_are_not_finite():
    rng = np.random.default_rng(2)
    c = Cache(2, 128, 64, True)
    x = rows_of(rng, 128, 2, 64)
    x[40, 0, 0] = np.nan
    x[90, 1, 5] = np.inf
    c.store(0, x, x)
    c.w.copy_(torch.arange(128.0).expand(2, 128))
    run_evict(c, 128, 60, 5)


# ---- together ----------------------------------------------------------------
def test_decode_with_a_budget():
    """A prompt, then tokens one by one; whenever the cache is full the heaviest rows move to the other one."""
    h, hq, d, budget, full = 2, 8, 64, 96, 160
    rng = np.random.default_rng(11)
    a, b = Cache(h, full, d, True, 1), Cache(h, full, d, True, 2)
    n = 0
    for step, n_new in enumerate([70, 40] + [1] * 60 + [9, 30] + [1] * 20):
        if n + n_new > full:
            kept = torch.empty(h, budget, dtype=torch.int32, device="cuda")
            a.q8.evict(n, budget, 32, b.q8, kept)
            for i in range(h):
                idx = kept[i].tolist()
                assert idx == R.evict(a.w[i].cpu().numpy(), n, budget, 32)
                for src, sw, dst, dw in zip(a.codes, a.words, b.codes, b.words):
                    x = R.row_values(src[i], sw[i])[idx]
                    for j in range(budget // B):
                        dst[i, j * B:(j + 1) * B], dw[i, j] = R.quantise_block(x[j * B:(j + 1) * B])
            b.check(budget)
            a, b, n = b, a, budget
        a.store(n, rows_of(rng, n_new, h, d), rows_of(rng, n_new, h, d))
        w0 = a.w.cpu().clone()
        check(a, hq, n, n_new, queries(step, n_new, hq, d), w0=w0)
        n += n_new
        a.check(n)


def test_captured_steps_replay():
    """store, attend, evict and load captured into a graph and replayed on other data, beside an eager run."""
    h, hq, d, n_past = 2, 8, 128, 1000
    c = filled(h, n_past, d, weight=True, extra=B * 2)
    c.w.uniform_()
    w0 = c.w.clone()
    new = [torch.zeros(2, h, d, device="cuda") for _ in range(2)]
    q = torch.zeros(2, hq * d, device="cuda")
    dst = Cache(h, 512, d, True)
    kept = torch.empty(h, 500, dtype=torch.int32, device="cuda")
    out, back = torch.empty(2, hq * d, device="cuda"), torch.empty(500, h, d, device="cuda")
    ws = torch.empty(c.q8.attend_workspace(hq, n_past, 2), dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream()
        c.q8.store(n_past, 2, *new, stream=s)
        c.q8.attend(hq, n_past, 2, q, out, workspace=ws, stream=s)
        c.q8.evict(n_past + 2, 500, 50, dst.q8, kept, stream=s)
        dst.q8.load(0, 500, back, None, stream=s)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        vals = [torch.randn(t.shape, generator=g) for t in (*new, q)]
        got = []
        for eager in (False, True):
            c.w.copy_(w0)
            for t, x in zip((*new, q), vals):
                t.copy_(x)
            if eager:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
            else:
                graph.replay()
            got.append([t.clone() for t in (out, back, kept, c.w)])
        assert all(torch.equal(x, y) for x, y in zip(*got))
        assert torch.isfinite(got[0][0]).all()


@pytest.mark.parametrize("n_new", [1, 5, 12, 40])
@pytest.mark.parametrize("size", [30000.0, 1.0, 1e-6])
def test_masked_blocks_in_which_nothing_was_stored(n_new, size):
    """Blocks whose codes and scale words are whatever the memory held, all of their keys masked with -inf."""
    h, hq, d, n_past = 40, 40, 64, 2000
    n_kv = n_past + n_new
    c = Cache(h, -(-n_kv // B) * B + B, d, weight=True)
    words = np.array([0, 0x7FFFFFFF, 0x7F800000, 0xFF800000, 0x80000000, 1, 0x7F7FFFFF, 0x7FC000E5, 0x00800000, 0xC1234567], np.uint32)
    rng = np.random.default_rng(3)
    mask = torch.zeros(n_new, n_kv)
    hidden = [b for b in range(n_past // B) if b % 3 == 1]
    for w, dw in zip(c.words, c.dev[2:]):
        for j, b in enumerate(hidden):
            w[:, b] = words[(np.arange(h) + j) % len(words)]
        dw.copy_(torch.from_numpy(w.view(np.float32)))
    for b in hidden:
        mask[:, b * B:(b + 1) * B] = float("-inf")
    at = 0
    for b in hidden + [None]:   # the rows between them, and the rest
        end = n_kv if b is None else b * B
        k = rng.standard_normal((end - at, h, d)).astype(np.float32)
        v = (rng.uniform(-1, 1, (end - at, h, d)) * size).astype(np.float32)
        c.store(at, k, v)
        at = n_kv if b is None else (b + 1) * B
    check(c, hq, n_past, n_new, queries(3, n_new, hq, d), mask=mask.cuda())


# ---- groups of more than 16 query heads ----------------------------------------
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("h, r, n_new, n_past", [(1, 17, 1, 0), (2, 33, 1, 500), (1, 71, 1, 90), (2, 71, 5, 700), (1, 100, 3, 333),
                                                 (1, 128, 1, 1000), (2, 128, 3, 64), (3, 65, 9, 1500)])
def test_attend_large_groups(d, h, r, n_new, n_past):
    """Tiles of 128 / r tokens with rows left over; rows of the weights' pass that are cut across tokens."""
    c = filled(h, n_past + n_new, d, weight=True, seed=n_past)
    c.w.uniform_(0.0, 2.0)
    check(c, h * r, n_past, n_new, queries(n_past, n_new, h * r, d), w0=c.w.cpu().clone())


@pytest.mark.parametrize("r, n_new", [(17, 1), (71, 2), (100, 4), (128, 1)])
@pytest.mark.parametrize("f16", [False, True])
def test_attend_large_groups_under_a_mask(r, n_new, f16):
    h, d, n_past = 2, 64, 300
    n_kv = n_past + n_new
    c = filled(h, n_kv, d, weight=True)
    mask = torch.randn(n_new, n_kv + 5, generator=torch.Generator().manual_seed(4))
    mask[torch.rand(mask.shape, generator=torch.Generator().manual_seed(5)) < 0.3] = float("-inf")
    if n_new > 1:
        mask[1] = float("-inf")
    mask = mask.to(torch.float16 if f16 else torch.float32).cuda()
    check(c, h * r, n_past, n_new, queries(9, n_new, h * r, d), mask=mask, flash=True)


def test_a_status_is_fine_after_calls_that_are():
    c = filled(2, 300, 64, weight=True)
    for n_new in (1, 40):
        check(c, 4, 300 - n_new, n_new, queries(1, n_new, 4, 64), w0=c.w.cpu().clone())
        assert c.q8.status() == K.KV_OK
        assert c.q8.status(torch.cuda.Stream()) == K.KV_OK


@pytest.mark.parametrize("n_new", [1, 3, 12, 40])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("size", [300.0, 3000.0, 30000.0])
def test_scores_of_any_size(n_new, masked, size):
    """Queries and keys up to F16's range: scores of up to 10^10, whose neighbours in 32 bits are far apart.  Values of
    different sizes from block to block, so that blocks have different exponents beside such a score.  Chunks without a mask
    are documented to hold scores of 10^7: a row with larger ones is right, or NaN and adds no weights."""
    h, hq, d, n_past = 2, 8, 64, 700
    n_kv, r = n_past + n_new, hq // h
    rng = np.random.default_rng(6)
    c = Cache(h, -(-n_kv // B) * B, d, weight=True)
    k = np.clip(rows_of(rng, n_kv, h, d) * size / 2, -60000, 60000)
    spread = np.repeat(2.0 ** rng.integers(-12, 12, n_kv // B + 1), B)[:n_kv, None, None]
    c.store(0, k.astype(np.float32), (rows_of(rng, n_kv, h, d) * spread).astype(np.float32))
    q = (queries(3, n_new, hq, d, f16=False) * size).clamp(-60000, 60000).half()
    mask = torch.zeros(n_new, n_kv).cuda() if masked else None
    kk = torch.from_numpy(np.stack([c.values(n_kv, i)[0].numpy() for i in range(h)]))
    vv = torch.from_numpy(np.stack([c.values(n_kv, i)[1].numpy() for i in range(h)]))
    s = torch.einsum("thrd,hnd->thrn", q.double().cpu().view(n_new, h, r, d), kk) / 8.0
    if not masked:
        s = s.masked_fill((torch.arange(n_kv)[None, :] > n_past + torch.arange(n_new)[:, None])[:, None, None, :], float("-inf"))
    far = s.nan_to_num(neginf=0.0).abs().amax(-1) > 1e7
    if masked or n_new * r <= 16 or not far.any():
        far = torch.zeros_like(far)
        out = check(c, hq, n_past, n_new, q, mask=mask)
    else:
        out = torch.zeros(n_new, hq * d, device="cuda")
        ws = torch.empty(c.q8.attend_workspace(hq, n_past, n_new), dtype=torch.uint8, device="cuda")
        c.q8.attend(hq, n_past, n_new, q, out, workspace=ws)
        # rows whose largest score has not passed 2^24 / log2(e), 1.17e7, by its exponent and rounding, add 1 each (a weight's
        # error is a factor of up to 2 there: an exponent's half step); no others do
        total = c.w.cpu().double().sum(-1)
        most = (s.amax(-1).abs() < 1.2e7).sum((0, 2)).double()
        assert torch.isfinite(c.w).all() and (total <= most * 2.0 + 1e-3).all() and (c.w >= 0).all()
    # all but the largest score's key is far below it: the outputs are its values
    top = s.topk(2, -1)
    # (the two largest apart by more than the sums' rounding, so that the second's weight is below 2^-24)
    err = (d + 4) * 2.0 ** -24 * s.abs().nan_to_num(posinf=0.0, neginf=0.0).amax(-1) * 4
    clear = top.values[..., 0] - top.values[..., 1] > 17.0 + err * 8
    want = torch.gather(vv[None].expand(n_new, -1, -1, -1), 2, top.indices[..., :1].expand(-1, -1, -1, d))
    got = out.double().cpu().view(n_new, h, r, d)
    assert clear.float().mean() > 0.5
    nan = torch.isnan(got).all(-1)
    assert not (nan & ~far).any() and torch.equal(nan, (~torch.isfinite(got)).any(-1))
    off = (got - want).abs() > want.abs() * 2.0 ** -10 + vv.abs().max() * 2.0 ** -23
    assert not (off.any(-1) & clear & ~nan).any()
