"""Cases of serving from a cache in 8 bits and of sampling a batch: rows stored
with a power-of-two scale for each block of tokens and head (and read back),
prompt and decode attention over such a cache, and a token drawn for each row of
logits by temperature, top-k, top-p and min-p.

`run` computes an operator in elementary torch operations (fp32; the sampler in
fp64, since a token changes where a sum crosses a border), or, where `own` is
true, by the calls of this library.  `exact` is the same definition in fp64,
sequence by sequence and row by row.
"""
import math

import torch

own = False

F32, F16 = 0, 1
TORCH = {"f32": torch.float32, "f16": torch.float16}
I8, F8 = 24, 64
KIND = {"i8": I8, "f8": F8}
TOP = {"i8": 127.0, "f8": 448.0}              # the largest number an element holds
LIMITS = {"i8": (-24, 9), "f8": (-15, 7)}     # exponents of a scale


def _ints(text):
    return [int(x) for x in str(text).split(",") if x != ""]


def _text(values):
    return ",".join(str(v) for v in values)


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one step of sixteen sequences: their keys and values into the cache,
        # most of them into blocks that hold rows already
        dict(name="append8 decode batch", op="append", lens=_text([1] * 16), hist=_text(range(5, 4005, 250)), heads=32,
             kv_heads=32, dim=128, src="f32", kv="i8", page=16, block=16),
        # three packed prompts, one of them continued
        dict(name="append8 packed prompts", op="append", lens="4096,2900,1195", hist="0,1111,0", heads=32, kv_heads=8,
             dim=128, src="f16", kv="f8", page=64, block=64),
        # the 128-token prompt of the 32-head decoder
        dict(name="prompt8 of 128 tokens", op="prompt", lens="128", hist="0", heads=32, kv_heads=32, dim=128, q="f32",
             kv="i8", page=16, block=16),
        # prompts of six users packed together
        dict(name="prompt8 packed fp16", op="prompt", lens="4096,1500,777,130,33,1", hist="0,0,0,0,0,0", heads=32,
             kv_heads=8, dim=128, q="f16", kv="f8", page=64, block=32),
        # a prompt taken in chunks behind a long history, and a short neighbour
        dict(name="prompt8 chunk with history", op="prompt", lens="511,64", hist="7001,300", heads=32, kv_heads=8,
             dim=128, q="f32", kv="i8", page=16, block=16),
        # one token of the small decoder: head dimension 48
        dict(name="decode8 one sequence", op="decode", lens="272", heads=6, kv_heads=6, dim=48, q="f32", kv="i8",
             page=32, block=32),
        # sixteen sequences of uneven age
        dict(name="decode8 batch of 16", op="decode",
             lens="4096,1,3900,260,2048,1777,95,3333,512,4001,1024,640,2900,16,1500,3584", heads=32, kv_heads=32,
             dim=128, q="f32", kv="i8", page=16, block=16),
        # few sequences, very long, grouped heads
        dict(name="decode8 long grouped", op="decode", lens="32768,30011,20480,9999", heads=32, kv_heads=8, dim=128,
             q="f16", kv="f8", page=64, block=64),
        # one user's token, the usual filters
        dict(name="sample one row", op="sample", rows=1, vocab=32000, logits="f32", spread=2.0, temperature=0.8,
             top_k=40, top_p=0.95, min_p=0.0, mixed=False),
        # a batch of sixteen, nucleus only
        dict(name="sample batch top-p", op="sample", rows=16, vocab=32000, logits="f32", spread=2.0, temperature=1.0,
             top_k=0, top_p=0.9, min_p=0.0, mixed=False),
        # every user has filters of their own, greedy ones among them; half-precision logits with many ties
        dict(name="sample mixed rows", op="sample", rows=33, vocab=50001, logits="f16", spread=2.5, temperature=0.9,
             top_k=0, top_p=1.0, min_p=0.0, mixed=True),
        # a large batch over a wide vocabulary, flat distributions
        dict(name="sample wide vocabulary", op="sample", rows=64, vocab=131072, logits="f32", spread=3.0,
             temperature=1.1, top_k=0, top_p=0.95, min_p=0.0, mixed=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


SHAPES = [(32, 32, 128), (32, 8, 128), (6, 6, 48), (8, 4, 32), (16, 2, 64), (16, 4, 96), (8, 1, 128), (12, 4, 80),
          (10, 2, 40)]


def draw(rng):
    op = rng.choice(["append", "prompt", "decode", "decode", "sample", "sample"])
    if op == "sample":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, vocab=_log(rng, 1000, 131072), logits=rng.choice(["f32", "f16"]),
                    spread=rng.choice([1.0, 2.0, 3.0]), temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, 0, _log(rng, 1, 2000)]), top_p=rng.choice([1.0, round(rng.uniform(0.2, 0.99), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]), mixed=rng.random() < 0.4)
    heads, kv_heads, dim = rng.choice(SHAPES)
    block = rng.choice([1, 16, 16, 32, 64])
    page = block * rng.choice([1, 2, 4]) if block > 1 else rng.choice([16, 24, 64])
    kv = rng.choice(["i8", "f8"])
    kind = rng.choice(["f32", "f16"])
    shape = dict(heads=heads, kv_heads=kv_heads, dim=dim, kv=kv, page=page, block=block)
    if op == "append":
        n = _log(rng, 1, 16)
        lens = [_log(rng, 1, 4096 // n) for _ in range(n)]
        return dict(op=op, lens=_text(lens), hist=_text(rng.randrange(0, 2000) for _ in range(n)), src=kind, **shape)
    if op == "prompt":
        n = _log(rng, 1, 6)
        lens = [_log(rng, 1, 3000) for _ in range(n)]
        return dict(op=op, lens=_text(lens), hist=_text(rng.choice([0, rng.randrange(0, 1000)]) for _ in range(n)),
                    q=kind, **shape)
    n = _log(rng, 1, 64)
    return dict(op=op, lens=_text(_log(rng, 1, 8192 if n <= 16 else 1024) for _ in range(n)), q=kind, **shape)


def _back(case):
    """Rows of each sequence that are read back after an append."""
    return [min(a + b, max(a, 16)) for a, b in zip(_ints(case["lens"]), _ints(case["hist"]))]


def work(case):
    size = {"f32": 4, "f16": 2}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["logits"]] + 32 * case["rows"], "flops": 10 * n}
    h, kh, d, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    lens = _ints(case["lens"])
    row = 2 * kh * d + 8 * kh / block               # a token's keys, values and share of the scales
    if case["op"] == "append":
        t, back = sum(lens), sum(_back(case))
        return {"bytes": t * (2 * kh * d * size[case["src"]] + row) + back * (row + 2 * kh * d * size[case["src"]]),
                "flops": 4 * (t + back) * kh * d}
    if case["op"] == "prompt":
        hist = _ints(case["hist"])
        seen = sum(n * b + n * (n + 1) // 2 for n, b in zip(lens, hist))
        return {"bytes": sum(lens) * h * d * 2 * size[case["q"]] + sum(n + b for n, b in zip(lens, hist)) * row,
                "flops": 4 * d * h * seen}
    return {"bytes": len(lens) * h * d * 2 * size[case["q"]] + sum(lens) * row, "flops": 4 * d * h * sum(lens)}


# --------------------------------------------------------------- the inputs

def _scale(amax, kind):
    """The least power of two with which `amax` fits, within the limits."""
    m, x = torch.frexp(amax)
    tm, tx = math.frexp(TOP[kind])
    e = x - tx + (m > tm).to(x.dtype)
    e = torch.where(amax == 0, torch.full_like(e, LIMITS[kind][0]), e).clamp(*LIMITS[kind])
    return torch.ldexp(torch.ones_like(amax), e)


def _held(x, scale, kind):
    """What a cache holds of x: elements of 8 bits."""
    y = x / scale
    if kind == "i8":
        return torch.round(y).clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _cache(case, g, counts):
    """A pool of normal values in 8 bits and a block table of shuffled pages
    with room for counts[i] rows of sequence i."""
    page, block, kh, d = case["page"], case["block"], case["kv_heads"], case["dim"]
    pages = [(c + page - 1) // page for c in counts]
    n_pages = sum(pages) + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(counts), max(1, max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = perm[at:at + p]
        at += p
    s = {"table": table}
    for name in ("k", "v"):
        x = torch.randn(n_pages * page // block, block, kh, d, generator=g, device="cuda")
        x *= torch.exp(0.5 * torch.randn(n_pages * page // block, 1, kh, 1, generator=g, device="cuda"))
        scale = _scale(x.abs().amax((1, 3)), case["kv"])
        s[name] = _held(x, scale[:, None, :, None], case["kv"]).view(n_pages, page, kh, d)
        s[name + "s"] = scale.view(n_pages, page // block, kh)
    return s


def _dev(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _packed(counts):
    return _dev([sum(counts[:i]) for i in range(len(counts) + 1)])


def _params(case, g):
    """Every row's temperature, top-k, top-p and min-p."""
    n = case["rows"]
    if not case["mixed"]:
        one = torch.ones(n, device="cuda")
        return one * case["temperature"], _dev([case["top_k"]] * n), one * case["top_p"], one * case["min_p"]

    def pick(values):
        return torch.tensor(values, device="cuda")[torch.randint(len(values), (n,), generator=g, device="cuda")]

    return (pick([0.0, 0.5, case["temperature"], 1.3]), pick([0, 0, 1, 40, 500]).to(torch.int32),
            pick([1.0, 0.5, 0.9, 0.99]), pick([0.0, 0.0, 0.02, 0.2]))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        # a bulk of unlikely tokens and a few dozen likely ones
        x = torch.randn(n, v, generator=g, device="cuda") * case["spread"]
        likely = torch.randint(v, (n, 40), generator=g, device="cuda")
        x.scatter_add_(1, likely, 3.0 + 3.0 * torch.randn(n, 40, generator=g, device="cuda").abs())
        t, k, p, m = _params(case, g)
        return {"case": case, "x": x.to(TORCH[case["logits"]]), "temperature": t, "top_k": k, "top_p": p, "min_p": m,
                "u": torch.rand(n, generator=g, device="cuda"),
                "token": torch.empty(n, dtype=torch.int32, device="cuda"), "prob": torch.empty(n, device="cuda"),
                "kept": torch.empty(n, dtype=torch.int32, device="cuda")}
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    lens = _ints(case["lens"])
    hist = _ints(case["hist"]) if "hist" in case else [0] * len(lens)
    both = [a + b for a, b in zip(lens, hist)]
    s = {"case": case, **_cache(case, g, both), "kv_len": _dev(both)}
    if case["op"] == "append":
        x = torch.randn(sum(lens), 2 * kh, d, generator=g, device="cuda").to(TORCH[case["src"]])
        s["kx"], s["vx"] = x[:, :kh], x[:, kh:]                   # one projection's rows
        s["cu"], s["cu_back"] = _packed(lens), _packed(_back(case))
        back = sum(_back(case))
        s["k_back"], s["v_back"] = (torch.empty(back, kh, d, dtype=x.dtype, device="cuda") for _ in range(2))
        return s
    tokens = len(lens) if case["op"] == "decode" else sum(lens)
    s["q"] = torch.randn(tokens, h, d, generator=g, device="cuda").to(TORCH[case["q"]])
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "prompt":
        s["cu"] = _packed(lens)
        s["max_q"], s["total_kv"] = max(lens), sum(both)
    s["max_kv"] = max(both)
    return s


# ----------------------------------------------------------- the plain form

def _tokens(cu, kv_len, total):
    """Sequence and slot of every packed row."""
    t = torch.arange(total, device="cuda")
    cu = cu.long()
    i = torch.searchsorted(cu, t, right=True) - 1
    return i, kv_len.long()[i] - cu[i + 1] + t


def _plain_append(s):
    case, page, block, kind = s["case"], s["case"]["page"], s["case"]["block"], s["case"]["kv"]
    kh, d = case["kv_heads"], case["dim"]
    seq, slot = _tokens(s["cu"], s["kv_len"], s["kx"].shape[0])
    at = s["table"][seq, slot // page].long()
    blk = at * (page // block) + slot % page // block             # the block of every new row
    own_blk, inv = torch.unique(blk, return_inverse=True)
    fresh = torch.zeros(own_blk.numel(), dtype=torch.bool, device="cuda")
    fresh[inv[slot % block == 0]] = True                          # its first row is new
    b_seq, b_slot = _tokens(s["cu_back"], s["kv_len"], s["k_back"].shape[0])
    b_at = s["table"][b_seq, b_slot // page].long()
    outs = []
    for name, x in (("k", s["kx"].float()), ("v", s["vx"].float())):
        pool, scales = s[name].view(-1, block, kh, d), s[name + "s"].view(-1, kh)
        amax = torch.zeros(own_blk.numel(), kh, device="cuda")
        amax.index_reduce_(0, inv, x.abs().amax(-1), "amax")
        old = scales[own_blk]
        need = _scale(amax, kind)
        now = torch.where(fresh[:, None], need, torch.maximum(need, old))
        had = pool[own_blk].float() * (torch.where(fresh[:, None], now, old) / now)[:, None, :, None]
        pool[own_blk] = _held(had, torch.ones_like(had[:1, :1, :1, :1]), kind)
        scales[own_blk] = now
        s[name][at, slot % page] = _held(x, scales[blk][:, :, None], kind)
        b_scale = scales[b_at * (page // block) + b_slot % page // block]
        outs.append((s[name][b_at, b_slot % page].float() * b_scale[:, :, None]).to(s["k_back"].dtype))
    return tuple(outs)


def _gather(s, name, rows):
    """Rows 0..rows-1 of every sequence, [sequences][kv heads][rows][dim] in fp32."""
    case = s["case"]
    t = s["table"][:, :(rows + case["page"] - 1) // case["page"]].long()
    x = s[name][t].float().flatten(1, 2)
    x *= s[name + "s"][t].flatten(1, 2).repeat_interleave(case["block"], 1)[..., None]
    return x[:, :rows].permute(0, 2, 1, 3)


def _plain_prompt(s):
    case, cu = s["case"], s["cu"].long()
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    lq, lk = s["max_q"], s["max_kv"]
    n, total = cu.numel() - 1, s["q"].shape[0]
    k, v = _gather(s, "k", lk), _gather(s, "v", lk)
    row = (cu[:-1, None] + torch.arange(lq, device="cuda")).clamp(max=total - 1)
    q = s["q"][row].float().view(n, lq, kh, h // kh, d).permute(0, 2, 3, 1, 4).reshape(n, kh, -1, d)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).view(n, h, lq, lk)
    kv_len = s["kv_len"].long()
    at = (kv_len - (cu[1:] - cu[:-1]))[:, None] + torch.arange(lq, device="cuda")
    seen = torch.arange(lk, device="cuda") <= at[:, :, None]
    x.masked_fill_(~seen[:, None], -math.inf)
    e = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(e.view(n, kh, -1, lk), v).view(n, h, lq, d) / e.sum(-1, keepdim=True)
    t = torch.arange(total, device="cuda")
    i = torch.searchsorted(cu, t, right=True) - 1
    return o[i, :, t - cu[i]].to(s["q"].dtype)


def _plain_decode(s):
    case = s["case"]
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    n, lk = s["q"].shape[0], s["max_kv"]
    q = s["q"].float().view(n, kh, h // kh, d)
    x = torch.matmul(q, _gather(s, "k", lk).transpose(-1, -2)) * d ** -0.5
    x.masked_fill_((torch.arange(lk, device="cuda") >= s["kv_len"].long()[:, None])[:, None, None], -math.inf)
    e = x.sub_(x.amax(-1, keepdim=True)).exp_()
    return (torch.matmul(e, _gather(s, "v", lk)) / e.sum(-1, keepdim=True)).reshape(n, h, d).to(s["q"].dtype)


def _plain_sample(s):
    x = s["x"].double()
    v = x.shape[1]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, t))
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where(k > 0, k, v))
    place = torch.arange(v, device="cuda")
    w.masked_fill_(place >= k, 0.0)
    sums = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    n = torch.minimum(k, (w >= s["min_p"].double()[:, None]).sum(1, keepdim=True))
    n = torch.where(p < 1, torch.minimum(n, 1 + (sums < p * sums[:, -1:]).sum(1, keepdim=True)), n)
    n = n.clamp(1, v)
    total = sums.gather(1, n - 1)
    at = (sums <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=n - 1)
    return (order.gather(1, at)[:, 0].int(), (w.gather(1, at) / total)[:, 0].float(), n[:, 0].int())


def _plain(s):
    return {"append": _plain_append, "prompt": _plain_prompt, "decode": _plain_decode,
            "sample": _plain_sample}[s["case"]["op"]](s)


# ------------------------------------------------------- the library's calls

def _rows(t):
    from tensoros_b200 import _ffi
    return _ffi.Rows(t.data_ptr(), t.stride(0), F32 if t.dtype == torch.float32 else F16)


def _bound(s):
    """The descriptors and the workspace that a user's program keeps for this
    shape, the calls made of them, and what they give."""
    import ctypes as C

    from tensoros_b200 import _ffi, lib
    case, L = s["case"], lib()
    keep = []

    def ref(x):
        keep.append(x)
        return C.byref(x)

    if case["op"] == "sample":
        params = ref(_ffi.SampleParams(s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(),
                                       s["min_p"].data_ptr()))
        args = (ref(_rows(s["x"])), case["rows"], case["vocab"], params, s["u"].data_ptr(), s["token"].data_ptr(),
                s["prob"].data_ptr(), s["kept"].data_ptr())
        return [(L.tos_sample_rows_dev, args)], (s["token"], s["prob"], s["kept"]), keep
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    kv = ref(_ffi.Paged8Kv(s["k"].data_ptr(), s["v"].data_ptr(), s["ks"].data_ptr(), s["vs"].data_ptr(),
                           KIND[case["kv"]], case["block"], s["k"].shape[0], case["page"], kh, d,
                           s["table"].data_ptr(), s["table"].shape[0], s["table"].stride(0)))
    n = s["kv_len"].numel()
    if case["op"] == "append":
        put = (kv, ref(_rows(s["kx"])), ref(_rows(s["vx"])), s["cu"].data_ptr(), s["kv_len"].data_ptr(), n,
               s["kx"].shape[0])
        get = (kv, ref(_rows(s["k_back"])), ref(_rows(s["v_back"])), s["cu_back"].data_ptr(), s["kv_len"].data_ptr(),
               n, s["k_back"].shape[0])
        return ([(L.tos_kv_append_paged8_dev, put), (L.tos_kv_read_paged8_dev, get)], (s["k_back"], s["v_back"]), keep)
    q, out, total = ref(_rows(s["q"])), ref(_rows(s["out"])), s["q"].shape[0]
    if case["op"] == "prompt":
        size = L.tos_attention_prompt_paged8_workspace_bytes(n, total, s["max_q"], s["total_kv"], s["max_kv"], h, kh, d)
    else:
        size = L.tos_attention_decode_paged8_workspace_bytes(n, s["max_kv"], h, kh, d)
    ws = torch.empty(max(size, 256), dtype=torch.uint8, device="cuda")
    keep.append(ws)
    if case["op"] == "prompt":
        args = (out, q, kv, s["cu"].data_ptr(), s["kv_len"].data_ptr(), n, total, s["max_q"], s["total_kv"],
                s["max_kv"], h, d ** -0.5, ws.data_ptr(), size)
        return [(L.tos_attention_prompt_paged8_dev, args)], s["out"], keep
    args = (out, q, kv, s["kv_len"].data_ptr(), n, s["max_kv"], h, d ** -0.5, ws.data_ptr(), size)
    return [(L.tos_attention_decode_paged8_dev, args)], s["out"], keep


def run(s):
    if not own:
        return _plain(s)
    if "calls" not in s:
        s["calls"] = _bound(s)
    calls, out, _ = s["calls"]
    # the library takes a null stream as its own; 1 is CUDA's legacy default stream
    stream = torch.cuda.current_stream().cuda_stream or 1
    for entry, args in calls:
        status = entry(*args, stream)
        if status:
            raise RuntimeError("%s: status %d" % (s["case"]["op"], status))
    return out


# ---------------------------------------------------- the definition in fp64

def _nearest(y, kind):
    """y rounded to the numbers that 8 bits hold, in fp64."""
    if kind == "i8":
        return torch.round(y).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_rows(s, name, i, n):
    """Rows 0..n-1 of sequence i in fp64, [n][kv heads][dim], and their scales."""
    page, block = s["case"]["page"], s["case"]["block"]
    j = torch.arange(n, device="cuda")
    at = s["table"][i].long()[j // page]
    scale = s[name + "s"][at, j % page // block].double()[:, :, None]
    return s[name][at, j % page].double() * scale, scale


def _exact_append(s):
    case, block, kind = s["case"], s["case"]["block"], s["case"]["kv"]
    lens, hist, back = _ints(case["lens"]), _ints(case["hist"]), _back(case)
    outs = []
    for name, src in (("k", s["kx"]), ("v", s["vx"])):
        got, at = [], 0
        for i, (n, b) in enumerate(zip(lens, hist)):
            x = src[at:at + n].double()
            at += n
            old, scale = _exact_rows(s, name, i, b)
            first = b // block * block
            rows = torch.cat([old[first:], x])
            new = torch.cat([torch.zeros_like(old[first:]), x]).abs().amax(-1)
            blocks = (rows.shape[0] + block - 1) // block
            pad = new.new_zeros(blocks * block, new.shape[1])
            pad[:new.shape[0]] = new
            amax = pad.view(blocks, block, -1).amax(1)
            # a logarithm may come out a hair above a whole number that it is; the next fp32 number is 8e-8 on
            e = torch.ceil(torch.log2(amax / TOP[kind]) - 1e-9).clamp(*LIMITS[kind])
            now = torch.exp2(e)
            if b % block:
                now[0] = torch.maximum(now[0], scale[first, :, 0])
            now = now.repeat_interleave(block, 0)[:rows.shape[0], :, None]
            both = torch.cat([old[:first], _nearest(rows / now, kind) * now])
            got.append(both[b + n - back[i]:])
        outs.append(torch.cat(got))
    return tuple(outs)


def _exact_attend(q, k, v, scale, last):
    """q [rows][dim], k and v [keys][dim] in fp64; row r sees keys 0..last[r]."""
    x = (q @ k.T) * scale
    x = torch.where(torch.arange(k.shape[0], device="cuda")[None] <= last[:, None], x, -math.inf)
    return torch.softmax(x, -1) @ v


def _exact_sample(s):
    outs = []
    for r in range(s["x"].shape[0]):
        x = s["x"][r].double()
        t, k, p, m = (float(s[c][r]) for c in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.argsort(x, descending=True, stable=True)
        w = torch.exp((x[order] - x.max()) / t) if t > 0 else (torch.arange(x.numel(), device="cuda") == 0).double()
        n = 1 if t <= 0 else min(int(k), x.numel()) if k > 0 else x.numel()
        sums = torch.cumsum(w[:n], 0)
        keep = n
        if p < 1:
            keep = min(keep, int(torch.searchsorted(sums, p * sums[-1])) + 1)
        keep = max(1, min(keep, int((w[:n] >= m).sum())))
        at = min(int(torch.searchsorted(sums[:keep], float(s["u"][r]) * sums[keep - 1], right=True)), keep - 1)
        outs.append((int(order[at]), float(w[at] / sums[keep - 1]), keep))
    token, prob, kept = zip(*outs)
    return (torch.tensor(token, dtype=torch.int32), torch.tensor(prob, dtype=torch.float64),
            torch.tensor(kept, dtype=torch.int32))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "append":
        return _exact_append(s)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    lens = _ints(case["lens"])
    decode = case["op"] == "decode"
    hist = [n - 1 for n in lens] if decode else _ints(case["hist"])
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, b in enumerate(hist):
        n = 1 if decode else lens[i]
        k, v = _exact_rows(s, "k", i, n + b)[0], _exact_rows(s, "v", i, n + b)[0]
        last = b + torch.arange(n, device="cuda")
        for j in range(h):
            out[at:at + n, j] = _exact_attend(s["q"][at:at + n, j].double(), k[:, j * kh // h], v[:, j * kh // h],
                                              d ** -0.5, last)
        at += n
    return out
