"""Long contexts in little memory, as cases that can be timed and checked.

Three operators, each through the calls that a serving engine makes of this package:

* ``write``: new K and V rows into a quantised cache, and the values it then holds of them back.
  An element is e4m3 ("fp8") or e2m1 ("fp4", two to a byte, the first in the low half); 32
  neighbouring elements of a head share a scale 2^(byte - 127), the smallest from 2^-100 to 2^118
  by which the largest of them fits.  ``read``: rows of such a cache over all its layers, as
  values of the model's type (an export of prompts).
* ``window``: attention over the paged cache in which a token sees itself, the `window` - 1
  tokens before it, and the first `sinks` tokens of its sequence.
* ``quant``: attention over a quantised paged cache, with a window or the whole context.

Head shapes are (query heads, KV heads, head_dim) of the Qwen2.5 / Qwen3 configurations that
the benchmark and the tests use, plus 256-wide heads.

Where `own` is false the operators are computed in elementary torch operations, batched over
sequences padded to the longest; where it is true, by the package's kernels.
"""

import math
from types import SimpleNamespace

import torch

own = False

BS = 16              # tokens per block
GROUP = 32           # elements that share a scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SHAPES = ((14, 2, 64), (12, 2, 128), (16, 8, 128), (28, 4, 128), (32, 8, 128))
PAIRS = 4 * 2048 * 32 * 8192          # sequences x queries x heads x keys of the largest case
KEYS = 16 * 32768 * 8 * 128           # cached numbers (of K) of the largest attention case
ROWS = 36 * 4096 * 8 * 128            # numbers (of K) of the largest write or read


# ------------------------------------------------------------------------------- the cases
def _rows(name, kind, layers, kv_heads, dim, tokens, fmt, dtype="bf16"):
    case = {"kind": kind, "layers": layers, "kv_heads": kv_heads, "dim": dim, "tokens": tokens,
            "fmt": fmt, "dtype": dtype}
    return {"name": name, **case} if name else case


def _attend(name, kind, shape, seqs, ctx, new, window, sinks, fmt="none", dtype="bf16", lengths=0):
    """seqs sequences of ctx[0]..ctx[1] tokens, of which the last new[0]..new[1] are queries; window
    0: the whole context.  The lengths follow from the number `lengths`."""
    case = {"kind": kind, "heads": shape[0], "kv_heads": shape[1], "dim": shape[2], "dtype": dtype,
            "fmt": fmt, "seqs": seqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "n_lo": new[0],
            "n_hi": new[1], "window": window, "sinks": sinks, "lengths": lengths}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one layer's new rows of a decoding batch: the smallest call, where launches count
        _rows("write_step", "write", 1, 8, 128, 32, "fp8"),
        # transferred prompts into every layer of the cache
        _rows("write_prompts", "write", 36, 8, 128, 2050, "fp8"),
        # a small model's prompt in a quarter of its size
        _rows("write_fp4", "write", 24, 2, 64, 777, "fp4", dtype="fp16"),
        # prompts read back for another worker
        _rows("read_prompts", "read", 36, 8, 128, 4096, "fp8"),
        # a few hundred tokens of an fp32 model
        _rows("read_fp4_fp32", "read", 24, 2, 64, 300, "fp4", dtype="fp32"),
        # a serving batch that streams: its last thousand tokens and four sinks
        _attend("window_decode", "window", (16, 8, 128), 32, (500, 8000), (1, 1), 1024, 4),
        # prompt chunks of long documents: the most arithmetic
        _attend("window_prefill", "window", (32, 8, 128), 4, (8192, 8192), (2048, 2048), 4096, 0),
        # verification of a few drafted tokens beside single ones
        _attend("window_verify_fp16", "window", (28, 4, 128), 24, (40, 3001), (1, 9), 512, 16,
                dtype="fp16"),
        # an fp32 model (reference-precision runs)
        _attend("window_fp32", "window", (14, 2, 64), 4, (200, 2000), (26, 26), 256, 4,
                dtype="fp32"),
        # long contexts decoded from half the bytes: the most memory
        _attend("quant_decode_long", "quant", (32, 8, 128), 16, (32768, 32768), (1, 1), 0, 0,
                fmt="fp8"),
        # prompt chunks behind contexts that are quantised already
        _attend("quant_prefill", "quant", (32, 8, 128), 4, (3000, 4608), (512, 512), 0, 0,
                fmt="fp8"),
        # a ragged batch in a quarter of the bytes, with window and sinks
        _attend("quant_window_fp4", "quant", (12, 2, 128), 48, (30, 6001), (1, 1), 2048, 4,
                fmt="fp4"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["write", "read", "window", "window", "quant", "quant"])
    if what in ("write", "read"):
        kv_heads, dim = rng.choice([(2, 64), (2, 128), (4, 128), (8, 128), (2, 256)])
        layers = rng.choice([1, rng.randint(2, 36)])
        most = max(1, ROWS // (layers * kv_heads * dim))
        return _rows(None, what, layers, kv_heads, dim, min(most, _log_int(rng, 1, 16384)),
                     rng.choice(["fp8", "fp8", "fp4"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    shape = rng.choice(SHAPES + ((8, 8, 256), (16, 8, 256)))
    small = dtype == "fp32"
    n_hi = rng.choice([1, _log_int(rng, 1, 32), _log_int(rng, 16, 256 if small else 2048)])
    ctx_hi = max(n_hi, _log_int(rng, 20, 4000 if small else 32768))
    seqs = _log_int(rng, 1, 16 if small else 64)
    seqs = max(1, min(seqs, PAIRS // (n_hi * shape[0] * ctx_hi), KEYS // (ctx_hi * shape[1] * shape[2])))
    n_hi = max(1, min(n_hi, PAIRS // (seqs * shape[0] * ctx_hi)))
    window = _log_int(rng, 16, 8192)
    if what == "quant" and rng.random() < 0.6:
        window = 0
    return _attend(None, what, shape, seqs, (rng.randint(1, ctx_hi), ctx_hi),
                   (rng.choice([n_hi, rng.randint(1, n_hi)]), n_hi), window,
                   rng.choice([0, 4, rng.randint(1, 64)]) if window else 0,
                   "none" if what == "window" else rng.choice(["fp8", "fp8", "fp4"]), dtype,
                   rng.randrange(1 << 30))


# ----------------------------------------------------------------------------- the inputs
def _lengths(case):
    """The numbers of new tokens of an attention case's sequences, and their context lengths."""
    g = torch.Generator().manual_seed(case["lengths"])

    def between(lo, hi):
        return torch.randint(lo, max(lo, hi) + 1, (case["seqs"],), generator=g).tolist()

    new, ctx = between(case["n_lo"], case["n_hi"]), between(case["ctx_lo"], case["ctx_hi"])
    new[-1] = case["n_hi"]
    ctx[0] = case["ctx_hi"]
    return new, [max(c, n) for c, n in zip(ctx, new)]


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _tables(lengths, g):
    """A block table of blocks in random places, and the pool's number of blocks."""
    need = [-(-n // BS) for n in lengths]
    perm = torch.randperm(sum(need) + 4, generator=g).to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32)
    for i, (n, at) in enumerate(zip(need, _cu(need))):
        table[i, :n] = perm[at:at + n]
    return table.cuda(), sum(need) + 4


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.Generator().manual_seed(seed + 1)
    s = SimpleNamespace(case=case, fmt=case["fmt"], dtype=DTYPES[case["dtype"]])
    return (_prepare_rows if case["kind"] in ("write", "read") else _prepare_attend)(case, s, gen, g)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _pool(gen, dim, *shape):
    """K or V rows: channels of unlike size."""
    return _randn(gen, *shape, dim) * _randn(gen, dim).mul_(0.5).exp_()


def _prepare_rows(case, s, gen, g):
    L, T, H, D = (case[x] for x in ("layers", "tokens", "kv_heads", "dim"))
    blocks = -(-T // BS) + 4
    table = torch.randperm(blocks, generator=g)
    pos = torch.arange(T)
    s.slots = (table[pos // BS] * BS + pos % BS).cuda()
    S = blocks * BS
    if case["kind"] == "write":
        s.k, s.v = (_pool(gen, D, L, T, H).to(s.dtype) for _ in "kv")
        shape = (L, S, H, D if s.fmt == "fp8" else D // 2)
        s.kc, s.vc = (torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in "kv")
        s.ks, s.vs = (torch.zeros((L, S, H, D // GROUP), dtype=torch.uint8, device="cuda")
                      for _ in "kv")
    else:
        # (layer by layer: little memory beside the pools)
        k, v = ([_encode(_pool(gen, D, S, H).to(s.dtype), s.fmt) for _ in range(L)] for _ in "kv")
        (s.kc, s.ks), (s.vc, s.vs) = ([torch.stack(t) for t in zip(*x)] for x in (k, v))
    return s


def _prepare_attend(case, s, gen, g):
    D, H = case["dim"], case["kv_heads"]
    s.new, s.ctx = _lengths(case)
    s.max_q, s.T = max(s.new), sum(s.new)
    s.cu_q, s.ctx_lens = _i32(_cu(s.new)), _i32(s.ctx)
    s.block_table, blocks = _tables(s.ctx, g)
    s.max_ctx = s.block_table.shape[1] * BS
    s.G, s.window, s.sinks = case["heads"] // H, case["window"], case["sinks"]
    s.q = _randn(gen, s.T, case["heads"], D).to(s.dtype)
    s.kc, s.vc = (_pool(gen, D, blocks * BS, H).to(s.dtype) for _ in "kv")
    if s.fmt != "none":
        (s.kc, s.ks), (s.vc, s.vs) = _encode(s.kc, s.fmt), _encode(s.vc, s.fmt)
    return s


# -------------------------------------------------------------- the formats, in plain form
def _encode(x, fmt):
    """Rows as codes and scales' bytes."""
    x = x.float() if x.dtype != torch.float16 else x.float().clamp(*_FP16[fmt])
    x = x.unflatten(-1, (-1, GROUP))
    top, least = (0.875, 9) if fmt == "fp8" else (0.75, 3)     # 448 and 6: top 2^least
    part, power = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(part <= top, power - least, power - least + 1)
    e = torch.where(part == 0, -100, e).clamp(-100, 118)
    largest = math.ldexp(top, least)
    y = torch.ldexp(x, -e).clamp(-largest, largest).flatten(-2)
    scale = (e[..., 0] + 127).to(torch.uint8)
    if fmt == "fp8":
        return y.to(torch.float8_e4m3fn).view(torch.uint8), scale
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step                           # (halves to the even code)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


# fp16 rows end where the next element up would be past fp16's largest number
_FP16 = {"fp8": (-61440.0, 61440.0), "fp4": (-49152.0, 49152.0)}


def _decode(code, scale, fmt):
    """The fp32 values that codes and scales' bytes stand for."""
    if fmt == "fp8":
        x = code.view(torch.float8_e4m3fn).float()
    else:
        half = torch.stack([code & 15, code >> 4], -1).flatten(-2).int()
        m, e = (half & 1).float(), (half >> 1) & 3
        x = torch.where(e == 0, 0.5 * m, torch.ldexp(1 + 0.5 * m, (e - 1).clamp(min=0)))
        x = torch.where(half >= 8, -x, x)
    power = (scale.int() - 127)[..., None]
    return torch.ldexp(x.unflatten(-1, (-1, GROUP)), power).flatten(-2)


# -------------------------------------------------------------------------------- the pass
def run(s):
    kind = s.case["kind"]
    if own:
        from dispec_amd.engine.hip_attn import paged_quant_attention, paged_window_attention
        from dispec_amd.kv.quant_cache import quant_append, quant_gather
        if kind == "write":
            quant_append(s.kc, s.ks, s.vc, s.vs, s.slots, s.k, s.v)
        if kind in ("write", "read"):
            return quant_gather(s.kc, s.ks, s.vc, s.vs, s.slots, s.dtype)
        more = dict(window=s.window, sinks=s.sinks, block_size=BS, max_q_len=s.max_q,
                    max_ctx=s.max_ctx)
        if kind == "quant":
            return paged_quant_attention(s.q, s.kc, s.ks, s.vc, s.vs, s.block_table, s.cu_q,
                                         s.ctx_lens, s.G, **more)
        return paged_window_attention(s.q, s.kc, s.vc, s.block_table, s.cu_q, s.ctx_lens, s.G, **more)
    if kind == "write":
        s.kc[:, s.slots], s.ks[:, s.slots] = _encode(s.k, s.fmt)
        s.vc[:, s.slots], s.vs[:, s.slots] = _encode(s.v, s.fmt)
    if kind in ("write", "read"):
        return (_decode(s.kc[:, s.slots], s.ks[:, s.slots], s.fmt).to(s.dtype),
                _decode(s.vc[:, s.slots], s.vs[:, s.slots], s.fmt).to(s.dtype))
    return _plain_attend(s)


def _plain_attend(s):
    B, (T, Hq, D), KVH, dev = len(s.new), s.q.shape, s.kc.shape[1], s.q.device
    n, C = s.max_q, s.max_ctx
    cu, ctx = s.cu_q.long(), s.ctx_lens.long()
    base = ctx - (cu[1:] - cu[:-1])
    query = torch.arange(n, device=dev)
    row = (cu[:-1, None] + query).clamp(max=T - 1)                     # (B, n)
    key = torch.arange(C, device=dev)
    slots = s.block_table.long()[:, key // BS] * BS + key % BS         # (B, C)
    k, v = s.kc[slots], s.vc[slots]
    if s.fmt != "none":
        k, v = _decode(k, s.ks[slots], s.fmt), _decode(v, s.vs[slots], s.fmt)
    # (B, KVH, D, C) keys, (B, KVH, C, D) values, (B, KVH, G n, D) queries
    k = k.float().permute(0, 2, 3, 1).contiguous()
    v = v.float().transpose(1, 2).contiguous()
    q = s.q[row].float().view(B, n, KVH, s.G, D).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, KVH, s.G * n, D)
    scores = torch.matmul(q, k).mul_(D ** -0.5).view(B, KVH, s.G, n, C)
    pos = (base[:, None] + query)[:, :, None]                          # (B, n, 1)
    hidden = key > pos
    if s.window:
        hidden = hidden | ((key <= pos - s.window) & (key >= s.sinks))
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KVH, s.G * n, C), v).view(B, KVH, s.G, n, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B * n, Hq, D)
    seq = torch.repeat_interleave(torch.arange(B, device=dev), cu[1:] - cu[:-1], output_size=T)
    return o[seq * n + torch.arange(T, device=dev) - cu[seq]].to(s.q.dtype)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    D = case["dim"]
    held = {"none": D * es, "fp8": D + D // GROUP, "fp4": D // 2 + D // GROUP}[case["fmt"]]
    if case["kind"] in ("write", "read"):
        rows = 2 * case["layers"] * case["tokens"] * case["kv_heads"]
        # (the codes out or in and the values out; written: the rows in too)
        wide = 2 if case["kind"] == "write" else 1
        return {"bytes": rows * (wide * D * es + held) + 8 * case["tokens"], "flops": 0}
    new, ctx = _lengths(case)
    W, S = case["window"], case["sinks"]
    pairs = keys = 0
    for n, c in zip(new, ctx):
        see = torch.arange(c - n + 1, c + 1, dtype=torch.int64)        # keys up to each query
        first = c - n + 1
        if W:
            see = see.clamp(max=W) + (see - W).clamp(min=0, max=S)
            first = min(first, W) + min(max(first - W, 0), S)
        pairs += int(see.sum())
        keys += first + n - 1
    T, Hq, H = sum(new), case["heads"], case["kv_heads"]
    return {"bytes": 2 * keys * H * held + 2 * T * Hq * D * es + keys / BS * 4,
            "flops": 4.0 * Hq * D * pairs}


# ------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return tuple(_nearest(x, s.fmt, s.dtype) for x in (s.k, s.v))
    if case["kind"] == "read":
        return tuple(_values(c[:, s.slots], e[:, s.slots], s.fmt)
                     for c, e in ((s.kc, s.ks), (s.vc, s.vs)))
    return _exact_attend(s)


def _numbers(fmt):
    """The numbers that an element's codes stand for."""
    bits, bias = (3, 7) if fmt == "fp8" else (1, 1)
    codes = range(128 if fmt == "fp8" else 8)
    return [math.ldexp(c % 2 ** bits + (2 ** bits if c >> bits else 0),
                       max(c >> bits, 1) - bias - bits) for c in codes]


def _values(code, scale, fmt):
    table = torch.tensor(_numbers(fmt), dtype=torch.float64, device="cuda")
    if fmt == "fp4":
        code = torch.stack([code % 16, code // 16], -1).flatten(-2)
    half = len(table)
    x = torch.cat([table, -table])[code.long() if half == 8 else code.long() % 256]
    return x * torch.exp2(scale.double() - 127).repeat_interleave(GROUP, -1)


def _nearest(x, fmt, dtype):
    """Each element's nearest number of its group's scale (the even code of two)."""
    numbers = _numbers(fmt)[:127 if fmt == "fp8" else 8]               # (127: no number)
    table = torch.tensor(numbers, dtype=torch.float64, device="cuda")
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for layer in range(x.shape[0]):
        y = x[layer].double().unflatten(-1, (-1, GROUP))
        if dtype == torch.float16:
            y = y.clamp(*_FP16[fmt])
        most = y.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(most / numbers[-1])).clamp(-100, 118)
        # (the logarithm may be off where it is nearly whole)
        e = e + (most > numbers[-1] * torch.exp2(e)).double()
        e = (e - (most <= numbers[-1] * torch.exp2(e - 1)).double()).clamp(-100, 118)
        a = (y.abs() / torch.exp2(e)).clamp(max=numbers[-1])
        up = torch.searchsorted(table, a.contiguous()).clamp(max=len(numbers) - 1)
        down = (up - 1).clamp(min=0)
        far, near = table[up] - a, a - table[down]
        pick = torch.where((far < near) | ((far == near) & (up % 2 == 0)), up, down)
        out[layer] = (table[pick] * torch.exp2(e) * torch.sign(y)).flatten(-2)
    return out


def _exact_attend(s):
    f, at = torch.float64, 0
    out = torch.empty(s.q.shape, dtype=f, device="cuda")
    for b, (n, c) in enumerate(zip(s.new, s.ctx)):
        pos = torch.arange(c, device="cuda")
        slots = s.block_table[b].long()[pos // BS] * BS + pos % BS
        query = torch.arange(c - n, c, device="cuda")[:, None]
        seen = pos <= query
        if s.window:
            seen &= (query - pos < s.window) | (pos < s.sinks)
        for h in range(s.kc.shape[1]):
            if s.fmt == "none":
                k, v = s.kc[slots, h].to(f), s.vc[slots, h].to(f)
            else:
                k = _values(s.kc[slots, h], s.ks[slots, h], s.fmt)
                v = _values(s.vc[slots, h], s.vs[slots, h], s.fmt)
            for j in range(h * s.G, (h + 1) * s.G):
                x = s.q[at:at + n, j].to(f) @ k.t().contiguous() / math.sqrt(s.q.shape[2])
                out[at:at + n, j] = x.masked_fill(~seen, -math.inf).softmax(-1) @ v
        at += n
    return out
