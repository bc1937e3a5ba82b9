"""The measured cases of the 8-bit KV cache: storing rows in it, reading them
back, attending over it (one token, several, a chunk; with and without the
accumulated attention weights) and evicting rows by those weights.

The cache of one layer: codes int8 [H][rows][D] for K and for V, one F32 scale
(a power of two) per KV head and block of 32 rows [H][rows/32], and F32
accumulated weights [H][rows].  A code c of block b stands for c * scale[b].

`own` false: the operators in elementary torch operations.  `own` true: the
library's entry points on the same buffers.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
DEV = "cuda"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decoded token's rows, in the middle of a block: the smallest call, latency
        dict(name="store-token", op="store", heads=8, dim=128, row0=1000, n_new=1, f16=False),
        # a 512-token chunk that starts and ends inside blocks
        dict(name="store-chunk", op="store", heads=8, dim=128, row0=16400, n_new=512, f16=True),
        # decode of a small model (14 query heads, 2 KV heads) near its 2k context
        dict(name="token-2k", op="attend", n_head=14, heads=2, dim=64, n_past=1999, n_new=1, mask="", weigh=False),
        # decode at a 32k context, 4 query heads a KV head
        dict(name="token-32k", op="attend", n_head=32, heads=8, dim=128, n_past=32100, n_new=1, mask="", weigh=False),
        # decode at a 128k context: the most bytes a call reads
        dict(name="token-128k", op="attend", n_head=32, heads=8, dim=128, n_past=131000, n_new=1, mask="", weigh=False),
        # a few draft tokens checked at once under the caller's mask, without grouped heads
        dict(name="draft-mask-4k", op="attend", n_head=32, heads=32, dim=96, n_past=4001, n_new=5, mask="f16", weigh=False),
        # a prompt's last, ragged chunk on an empty cache
        dict(name="prompt-small", op="attend", n_head=14, heads=2, dim=64, n_past=0, n_new=257, mask="", weigh=False),
        # a full chunk deep in a prompt: the most arithmetic a call does
        dict(name="chunk-16k", op="attend", n_head=32, heads=8, dim=128, n_past=16384, n_new=512, mask="", weigh=False),
        # decode that accumulates the weights an eviction goes by
        dict(name="token-32k-weigh", op="attend", n_head=32, heads=8, dim=128, n_past=32100, n_new=1, mask="", weigh=True),
        # a prompt chunk that accumulates them
        dict(name="chunk-4k-weigh", op="attend", n_head=32, heads=8, dim=128, n_past=4096, n_new=512, mask="", weigh=True),
        # a short cache halved
        dict(name="evict-2k", op="evict", heads=2, dim=64, n_rows=2047, keep=1023, recent=127),
        # a long cache halved
        dict(name="evict-32k", op="evict", heads=8, dim=128, n_rows=32700, keep=16384, recent=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dim = rng.choice([64, 96, 128, 128, 256])
    heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    kind = rng.choice(["store", "token", "token", "few", "chunk", "chunk", "evict"])
    if kind == "store":
        return dict(op="store", heads=heads, dim=dim, row0=_log(rng, 1, 30000) - 1, n_new=_log(rng, 1, 512),
                    f16=rng.random() < 0.5)
    if kind == "evict":
        n = min(_log(rng, 64, 60000), 32700 * 8 * 128 // (heads * dim))
        keep = max(1, int(n * rng.uniform(0.1, 0.95)))
        return dict(op="evict", heads=heads, dim=dim, n_rows=n, keep=keep, recent=int(keep * rng.uniform(0.0, 0.6)))
    group = rng.choice([1, 2, 4, 4, 5, 7, 8])
    n_new = 1 if kind == "token" else _log(rng, 2, 16) if kind == "few" else _log(rng, 17, 512)
    most = 131000 * 8 * 128 // (heads * dim)                         # the bytes of token-128k
    if kind != "token":
        most = min(most, 16384 * 512 * 32 * 128 // (n_new * heads * group * dim))   # the products of chunk-16k
    n_past = min(_log(rng, rng.choice([1, 256, 2048]), 131000) - 1, max(0, most - n_new))
    small = n_new * (n_past + n_new) <= 4 << 20
    return dict(op="attend", n_head=heads * group, heads=heads, dim=dim, n_past=n_past, n_new=n_new,
                mask=rng.choice(["", "", "f16", "f32"]) if small else "", weigh=rng.random() < 0.35)


def _blocks(rows):
    return -(-rows // BLOCK)


def _touched(case):
    """The stored rows and those of their first block before them: [first, end)."""
    return case["row0"] // BLOCK * BLOCK, case["row0"] + case["n_new"]


def work(case):
    h, d = case["heads"], case["dim"]
    if case["op"] == "store":
        first, end = _touched(case)
        new, old = case["n_new"], case["row0"] - first
        # the new rows read, the block's earlier codes read, the new codes written, all of them read back as F16
        return {"bytes": 2 * h * d * (new * (2 if case["f16"] else 4) + old + new + (end - first) * 2), "flops": 0}
    if case["op"] == "evict":
        n, keep = case["n_rows"], case["keep"]
        # the weights read; the kept codes read and written; their weights and places written; their values read back
        return {"bytes": h * (4 * n + 8 * keep + 2 * keep * d * (1 + 1 + 2)), "flops": 0}
    n_new, n_kv, hq = case["n_new"], case["n_past"] + case["n_new"], case["n_head"]
    size = {"": 0, "f16": 2, "f32": 4}[case["mask"]]
    bytes_ = 2 * h * (n_kv * d + 4 * _blocks(n_kv)) + n_new * hq * d * 4 + size * n_new * n_kv
    if case["weigh"]:
        bytes_ += 8 * h * n_kv
    seen = n_new * n_kv if case["mask"] else n_new * case["n_past"] + n_new * (n_new + 1) // 2
    return {"bytes": bytes_, "flops": 4 * d * hq * seen}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rows(gen, heads, n, dim, dtype=torch.float32):
    """Rows as a projection gives them: a few channels larger than the others, tokens of different size, a mean."""
    x = torch.randn(heads, n, dim, generator=gen, device=DEV, dtype=dtype)
    gain = torch.rand(heads, 1, dim, generator=gen, device=DEV).pow(8).mul_(2.0).add_(0.7)
    size = torch.randn(heads, n, 1, generator=gen, device=DEV).mul_(0.25).exp_()
    return x.mul_(gain.to(dtype)).mul_(size.to(dtype)).add_(0.1)


def _cache(gen, heads, rows, dim):
    """A filled cache of `rows` rows (a multiple of the block)."""
    out = []
    for _ in range(2):
        codes, scale = _quantise(_rows(gen, heads, rows, dim).half().float())
        out += [codes, scale]
    return dict(k=out[0], v=out[2], k_scale=out[1], v_scale=out[3])


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    h, d = case["heads"], case["dim"]
    s = dict(case=dict(case))
    if case["op"] == "store":
        first, end = _touched(case)
        s.update(_cache(gen, h, _blocks(end) * BLOCK + BLOCK, d))
        dtype = torch.float16 if case["f16"] else torch.float32
        # K and V as they lie in one fused row of a projection
        fused = torch.cat([_rows(gen, h, case["n_new"], d), _rows(gen, h, case["n_new"], d)])
        fused = fused.transpose(0, 1).reshape(case["n_new"], 2 * h * d).to(dtype).contiguous()
        s.update(new_k=fused[:, :h * d], new_v=fused[:, h * d:])
        return s
    if case["op"] == "evict":
        n, keep = case["n_rows"], case["keep"]
        s.update(_cache(gen, h, _blocks(n) * BLOCK, d))
        # a few heavy rows, many light ones, and some that no query looked at: equal weights
        w = torch.randn(h, _blocks(n) * BLOCK, generator=gen, device=DEV).mul_(2.0).exp_()
        w[torch.rand(w.shape, generator=gen, device=DEV) < 0.2] = 0.0
        s["weight"] = w
        kr = _blocks(keep) * BLOCK
        s.update(dst_k=torch.zeros(h, kr, d, dtype=torch.int8, device=DEV),
                 dst_v=torch.zeros(h, kr, d, dtype=torch.int8, device=DEV),
                 dst_k_scale=torch.ones(h, kr // BLOCK, device=DEV), dst_v_scale=torch.ones(h, kr // BLOCK, device=DEV),
                 dst_weight=torch.zeros(h, kr, device=DEV), kept=torch.zeros(h, keep, dtype=torch.int32, device=DEV))
        return s
    n_new, n_kv, hq = case["n_new"], case["n_past"] + case["n_new"], case["n_head"]
    s.update(_cache(gen, h, _blocks(n_kv) * BLOCK + BLOCK, d))   # the last block holds nothing that is attended
    q = torch.randn(n_new, hq * d + 2 * h * d, generator=gen, device=DEV).mul_(1.2).half()
    s["q"] = q[:, :hq * d]                                       # the Q part of fused Q/K/V rows
    s["weight"] = torch.rand(h, s["k"].shape[1], generator=gen, device=DEV) if case["weigh"] else None
    s["mask"] = None
    if case["mask"]:
        # a draft's mask: the past, oneself and some of the other new tokens; a few past keys removed, a bias on the rest
        m = torch.randn(n_new, n_kv, generator=gen, device=DEV).mul_(0.5)
        m[torch.rand(m.shape, generator=gen, device=DEV) < 0.1] = float("-inf")
        new = torch.rand(n_new, n_new, generator=gen, device=DEV) < 0.5
        new = torch.tril(new, -1) | torch.eye(n_new, dtype=torch.bool, device=DEV)
        m[:, case["n_past"]:] = torch.zeros(n_new, n_new, device=DEV).masked_fill_(~new, float("-inf"))
        s["mask"] = m.to(torch.float16 if case["mask"] == "f16" else torch.float32)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _exponent(amax):
    """The smallest e in [-24, 9] for which amax / 2^e rounds to at most 127."""
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -24).double())) - 6
    e = torch.where(torch.round(amax.double() * torch.exp2(-e)) > 127, e + 1, e)
    return e.clamp(-24, 9)


def _quantise(x):
    """Codes and scales of whole blocks: x [H][rows][D], finite values that F16 holds."""
    h, rows, d = x.shape
    e = _exponent(x.view(h, rows // BLOCK, BLOCK * d).abs().amax(-1))
    scale = torch.exp2(e).float()
    codes = torch.round(x.view(h, rows // BLOCK, BLOCK, d) / scale[:, :, None, None]).clamp_(-127, 127)
    return codes.to(torch.int8).view(h, rows, d), scale


def _values(codes, scale, rows):
    """What the first `rows` rows stand for, F32 [H][rows][D]."""
    return codes[:, :rows].float() * scale.repeat_interleave(BLOCK, 1)[:, :rows, None]


def _plain_store(s):
    case = s["case"]
    h, d = case["heads"], case["dim"]
    first, end = _touched(case)
    last = _blocks(end) * BLOCK
    got = []
    for codes, scale, new in ((s["k"], s["k_scale"], s["new_k"]), (s["v"], s["v_scale"], s["new_v"])):
        x = torch.zeros(h, last - first, d, device=DEV)
        old = case["row0"] - first
        x[:, :old] = _values(codes[:, first:last], scale[:, first // BLOCK:], old)
        x[:, old:end - first] = new.half().float().view(case["n_new"], h, d).transpose(0, 1)
        c, sc = _quantise(x)
        codes[:, first:end] = c[:, :end - first]
        scale[:, first // BLOCK:last // BLOCK] = sc
        got.append(_values(c, sc, end - first).transpose(0, 1).half().contiguous())
    return got


def _scores(s):
    """Scaled scores with the mask, F32 [H][n_new][group][n_kv]."""
    case = s["case"]
    h, d, n_new, n_kv = case["heads"], case["dim"], case["n_new"], case["n_past"] + case["n_new"]
    k = _values(s["k"], s["k_scale"], n_kv)
    q = s["q"].float().view(n_new, h, -1, d).transpose(0, 1)
    t = torch.matmul(q.reshape(h, -1, d), k.transpose(1, 2)).mul_(1.0 / math.sqrt(d)).view(h, n_new, -1, n_kv)
    if s["mask"] is not None:
        return t.add_(s["mask"].float()[None, :, None, :])
    at = torch.arange(n_kv, device=DEV)
    hidden = at[None, :] > case["n_past"] + torch.arange(n_new, device=DEV)[:, None]
    return t.masked_fill_(hidden[None, :, None, :], float("-inf"))


def _plain_attend(s):
    case = s["case"]
    h, d, n_new, n_kv = case["heads"], case["dim"], case["n_new"], case["n_past"] + case["n_new"]
    p = _scores(s)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p.view(h, -1, n_kv), _values(s["v"], s["v_scale"], n_kv))
    out = o.view(h, n_new, -1, d).transpose(0, 1).reshape(n_new, case["n_head"] * d).half()
    if s["weight"] is None:
        return out
    s["weight"][:, :n_kv] += p.sum((1, 2))
    return out, s["weight"]


def _plain_evict(s):
    case = s["case"]
    n, keep, recent = case["n_rows"], case["keep"], case["recent"]
    order = torch.sort(s["weight"][:, :n - recent], dim=1, descending=True, stable=True).indices[:, :keep - recent]
    last = torch.arange(n - recent, n, device=DEV).expand(order.shape[0], recent)
    kept = torch.cat([order.sort(1).values, last], 1)
    rows = _blocks(keep) * BLOCK
    got = []
    for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = torch.gather(_values(codes, scale, n), 1, kept[:, :, None].expand(-1, -1, codes.shape[2]))
        x = torch.cat([x, x.new_zeros(x.shape[0], rows - keep, x.shape[2])], 1)
        got.append(_values(*_quantise(x), keep).transpose(0, 1).half().contiguous())
    return got[0], got[1], torch.gather(s["weight"], 1, kept), kept.int()


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _handle(s):
    """The views of the buffers and the workspace that a program keeps from one call to the next."""
    if "handle" not in s:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ggml-loader_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import kv_b200
        case = s["case"]
        cache = kv_b200.Q8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], s.get("weight"))
        more = None
        if case["op"] == "evict":
            more = kv_b200.Q8Cache(s["dst_k"], s["dst_v"], s["dst_k_scale"], s["dst_v_scale"], s["dst_weight"])
        elif case["op"] == "attend":
            more = torch.empty(cache.attend_workspace(case["n_head"], case["n_past"], case["n_new"]),
                               dtype=torch.uint8, device=DEV)
        s["handle"] = cache, more
    return s["handle"]


def _own_run(s):
    case = s["case"]
    h, d = case["heads"], case["dim"]
    cache, more = _handle(s)
    stream = torch.cuda.current_stream()
    if case["op"] == "attend":
        out = torch.empty(case["n_new"], case["n_head"] * d, dtype=torch.float16, device=DEV)
        cache.attend(case["n_head"], case["n_past"], case["n_new"], s["q"], out, mask=s["mask"], workspace=more,
                     stream=stream)
        return out if s["weight"] is None else (out, s["weight"])
    if case["op"] == "store":
        cache.store(case["row0"], case["n_new"], s["new_k"], s["new_v"], stream=stream)
        first, end = _touched(case)
        back = cache
    else:
        cache.evict(case["n_rows"], case["keep"], case["recent"], more, s["kept"], stream=stream)
        first, end, back = 0, case["keep"], more
    k = torch.empty(end - first, h, d, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    back.load(first, end - first, k, v, stream=stream)
    return [k, v] if case["op"] == "store" else (k, v, s["dst_weight"][:, :end], s["kept"])


def run(state):
    if own:
        return _own_run(state)
    return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_block(x):
    """What a block of values is stored as, in 64 bits: the first exponent, from below, at which none rounds past 127."""
    top = float(x.abs().max()) if x.numel() else 0.0
    e = -24
    while e < 9 and round(top / 2.0 ** e) > 127:
        e += 1
    return torch.clamp(torch.round(x * 2.0 ** -e), -127, 127) * 2.0 ** e


def _exact_blocks(x):
    """x [H][rows][D] in 64 bits, blocks counted from its first row."""
    y = x.cpu()
    return torch.stack([torch.cat([_exact_block(y[i, b:b + BLOCK]) for b in range(0, y.shape[1], BLOCK)])
                        for i in range(y.shape[0])])


def _exact_values(codes, scale):
    rows = torch.arange(codes.shape[1], device=DEV) // BLOCK
    return codes.double() * scale.double()[:, rows].unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    h, d = case["heads"], case["dim"]
    if case["op"] == "store":
        first, end = _touched(case)
        got = []
        for codes, scale, new in ((s["k"], s["k_scale"], s["new_k"]), (s["v"], s["v_scale"], s["new_v"])):
            old = _exact_values(codes, scale)[:, first:case["row0"]]
            new = new.half().double().reshape(case["n_new"], h, d).permute(1, 0, 2)
            got.append(_exact_blocks(torch.cat([old, new], 1)).permute(1, 0, 2).contiguous())
        return got
    if case["op"] == "evict":
        n, keep, recent = case["n_rows"], case["keep"], case["recent"]
        w = s["weight"].double().cpu()
        kept = []
        for i in range(h):
            heavy = sorted(range(n - recent), key=w[i].tolist().__getitem__, reverse=True)[:keep - recent]
            kept.append(sorted(heavy) + list(range(n - recent, n)))
        kept = torch.tensor(kept, dtype=torch.int64)
        got = []
        for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
            x = _exact_values(codes, scale).cpu()
            x = torch.stack([x[i, kept[i]] for i in range(h)])
            got.append(_exact_blocks(x).permute(1, 0, 2).contiguous())
        return got[0], got[1], torch.stack([w[i, kept[i]] for i in range(h)]), kept.int()
    n_new, n_past, hq = case["n_new"], case["n_past"], case["n_head"]
    n_kv, group = n_past + n_new, hq // h
    out = torch.empty(n_new, hq, d, dtype=torch.float64, device=DEV)
    weight = None if s["weight"] is None else s["weight"].double()
    k, v = _exact_values(s["k"], s["k_scale"])[:, :n_kv], _exact_values(s["v"], s["v_scale"])[:, :n_kv]
    bias = torch.zeros(n_new, n_kv, dtype=torch.float64, device=DEV)
    if s["mask"] is not None:
        bias += s["mask"].double()
    else:
        for t in range(n_new):
            bias[t, n_past + t + 1:] = float("-inf")
    q = s["q"].double().reshape(n_new, hq, d)
    for j in range(hq):
        t = q[:, j] @ k[j // group].T / math.sqrt(d) + bias
        p = torch.exp(t - torch.logsumexp(t, 1, keepdim=True))
        out[:, j] = p @ v[j // group]
        if weight is not None:
            weight[j // group, :n_kv] += p.sum(0)
    out = out.reshape(n_new, hq * d)
    return out if weight is None else (out, weight)
