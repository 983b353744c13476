"""Cases of the paged-cache operators: per-head norm and rotary positions, the
append to the paged cache, prompt attention over packed sequences and decode
attention with a shared prefix.

`run` computes an operator in elementary torch operations (fp32, angles in
fp64), or, where `own` is true, by the calls of this library.  `exact` is the
same definition in fp64, sequence by sequence and head by head.
"""
import math

import torch

own = False

F32, F16 = 0, 1
TORCH = {"f32": torch.float32, "f16": torch.float16}
CODE = {"f32": F32, "f16": F16}
EPS = 1e-6
BASE = 10000.0
ORIG_CTX = 4096
BETA_FAST, BETA_SLOW = 32.0, 1.0


def _ints(text):
    return [int(x) for x in str(text).split(",") if x != ""]


def _text(values):
    return ",".join(str(v) for v in values)


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one decoded token of the 32-head, 128-wide decoder between its
        # fp32 projections and a cache the caller keeps himself
        dict(name="rotary one token", op="rotary", tokens=1, heads=32, kv_heads=32, dim=128, src="f32", dst="f32",
             rot=128, layout="interleaved", scaling="none", factor=1.0, norm=False, first=777),
        # a long prompt of a grouped-query model with normalised heads whose
        # context is stretched four times
        dict(name="rotary norm long prompt", op="rotary", tokens=4099, heads=32, kv_heads=8, dim=128, src="f16",
             dst="f16", rot=128, layout="half", scaling="yarn", factor=4.0, norm=True, first=12288),
        # a prompt whose heads rotate in part, narrowed to fp16 on the way
        dict(name="rotary part of the head", op="rotary", tokens=2047, heads=16, kv_heads=2, dim=64, src="f32",
             dst="f16", rot=32, layout="half", scaling="linear", factor=2.0, norm=False, first=0),
        # one step of a batch of sixteen sequences: fp32 projections into an
        # fp16 cache, q rotated in the same call
        dict(name="append decode batch", op="append", lens=_text([1] * 16), hist=_text(range(5, 4005, 250)), heads=32,
             kv_heads=32, dim=128, src="f32", kv="f16", page=16, rot=128, layout="interleaved", scaling="none",
             factor=1.0, norm=False),
        # three packed prompts, one of them continued, into 64-token pages
        dict(name="append packed prompts", op="append", lens="4096,2900,1195", hist="0,1111,0", heads=32, kv_heads=8,
             dim=128, src="f16", kv="f16", page=64, rot=128, layout="half", scaling="none", factor=1.0, norm=True),
        # the 128-token prompt of the 32-head decoder
        dict(name="prompt of 128 tokens", op="prompt", lens="128", hist="0", heads=32, kv_heads=32, dim=128, q="f32",
             kv="f16", page=16),
        # prompts of six users packed together, all in half precision
        dict(name="prompt packed fp16", op="prompt", lens="4096,1500,777,130,33,1", hist="0,0,0,0,0,0", heads=32,
             kv_heads=8, dim=128, q="f16", kv="f16", page=64),
        # a prompt taken in chunks: 511 new tokens behind a long history, and
        # a short neighbour
        dict(name="prompt chunk with history", op="prompt", lens="511,64", hist="7001,300", heads=32, kv_heads=8,
             dim=128, q="f32", kv="f16", page=16),
        # the small fp32 decoder's prompt: head dimension 48, fp32 cache
        dict(name="prompt small fp32", op="prompt", lens="272,16", hist="0,0", heads=6, kv_heads=6, dim=48, q="f32",
             kv="f32", page=32),
        # one token of the small fp32 decoder
        dict(name="decode one fp32", op="decode", lens="272", prefix=0, heads=6, kv_heads=6, dim=48, q="f32",
             kv="f32", page=32),
        # sixteen sequences of uneven age
        dict(name="decode batch of 16", op="decode",
             lens="4096,1,3900,260,2048,1777,95,3333,512,4001,1024,640,2900,16,1500,3584", prefix=0, heads=32,
             kv_heads=32, dim=128, q="f32", kv="f16", page=16),
        # sixty-four answers to one long document
        dict(name="decode shared prefix", op="decode", lens=_text(1 + (i * 197) % 512 for i in range(64)), prefix=8190,
             heads=32, kv_heads=8, dim=128, q="f16", kv="f16", page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


SHAPES = [(32, 32, 128), (32, 8, 128), (6, 6, 48), (8, 4, 32), (16, 2, 64), (16, 4, 96), (8, 1, 128), (12, 4, 80)]


def draw(rng):
    heads, kv_heads, dim = rng.choice(SHAPES)
    op = rng.choice(["rotary", "append", "prompt", "prompt", "decode", "decode"])
    page = rng.choice([16, 32, 64, 128])
    rotary = dict(rot=rng.choice([dim, dim, dim // 2]), layout=rng.choice(["interleaved", "half"]),
                  scaling=rng.choice(["none", "linear", "yarn"]), norm=rng.random() < 0.5)
    rotary["factor"] = 1.0 if rotary["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0])
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, 4096), heads=heads, kv_heads=kv_heads, dim=dim,
                    src=rng.choice(["f32", "f16"]), dst=rng.choice(["f32", "f16"]), first=_log(rng, 1, 100000),
                    **rotary)
    if op == "append":
        n = _log(rng, 1, 16)
        lens = [_log(rng, 1, 4096 // n) for _ in range(n)]
        return dict(op=op, lens=_text(lens), hist=_text(rng.randrange(0, 2000) for _ in range(n)), heads=heads,
                    kv_heads=kv_heads, dim=dim, src=rng.choice(["f32", "f16"]), kv=rng.choice(["f16", "f16", "f32"]),
                    page=page, **rotary)
    kind = rng.choice([("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
    if op == "prompt":
        n = _log(rng, 1, 6)
        most = 1024 if kind[1] == "f32" else 3000
        lens = [_log(rng, 1, most) for _ in range(n)]
        return dict(op=op, lens=_text(lens), hist=_text(rng.choice([0, rng.randrange(0, 1000)]) for _ in range(n)),
                    heads=heads, kv_heads=kv_heads, dim=dim, q=kind[0], kv=kind[1], page=page)
    n = _log(rng, 1, 64)
    return dict(op=op, lens=_text(_log(rng, 1, 4096 if n <= 16 else 1024) for _ in range(n)),
                prefix=rng.choice([0, _log(rng, 1, 8190)]), heads=heads, kv_heads=kv_heads, dim=dim, q=kind[0],
                kv=kind[1], page=page)


def work(case):
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    size = {"f32": 4, "f16": 2}
    if case["op"] == "rotary":
        n = case["tokens"] * (h + kh) * d
        return {"bytes": n * (size[case["src"]] + size[case["dst"]]) + 4 * case["tokens"], "flops": 8 * n}
    if case["op"] == "append":
        t = sum(_ints(case["lens"]))
        return {"bytes": t * d * (h * 2 * size[case["src"]] + 2 * kh * (size[case["src"]] + size[case["kv"]])) + 12 * t,
                "flops": 8 * t * (h + kh) * d}
    if case["op"] == "prompt":
        lens, hist = _ints(case["lens"]), _ints(case["hist"])
        seen = sum(n * b + n * (n + 1) // 2 for n, b in zip(lens, hist))
        rows = sum(n + b for n, b in zip(lens, hist))
        return {"bytes": sum(lens) * h * d * 2 * size[case["q"]] + rows * kh * d * 2 * size[case["kv"]],
                "flops": 4 * d * h * seen}
    lens = _ints(case["lens"])
    return {"bytes": len(lens) * h * d * 2 * size[case["q"]] + (sum(lens) + case["prefix"]) * kh * d * 2 * size[case["kv"]],
            "flops": 4 * d * h * (sum(lens) + len(lens) * case["prefix"])}


# --------------------------------------------------------------- the inputs

def _cache(case, g, counts):
    """A cache of normal values and a block table of shuffled pages with room
    for counts[i] rows of sequence i."""
    page, kh, d = case["page"], case["kv_heads"], case["dim"]
    pages = [(c + page - 1) // page for c in counts]
    n_pages = sum(pages) + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(counts), max(1, max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = perm[at:at + p]
        at += p
    kc = torch.randn(n_pages, page, kh, d, generator=g, device="cuda").to(TORCH[case["kv"]])
    vc = torch.randn(n_pages, page, kh, d, generator=g, device="cuda").to(TORCH[case["kv"]])
    return kc, vc, table


def _dev(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}

    def rand(*shape, kind):
        return torch.randn(*shape, generator=g, device="cuda").to(TORCH[kind])

    def weights():
        if case["norm"]:
            s["qw"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
            s["kw"] = 1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")
        else:
            s["qw"] = s["kw"] = None

    if case["op"] == "rotary":
        n = case["tokens"]
        s["qkv"] = rand(n, h + kh, d, kind=case["src"])     # one projection's rows: q heads, then k heads
        s["q"], s["k"] = s["qkv"][:, :h], s["qkv"][:, h:]
        s["pos"] = (case["first"] + torch.arange(n, device="cuda")).to(torch.int32)
        s["q_out"] = torch.empty(n, h, d, dtype=TORCH[case["dst"]], device="cuda")
        s["k_out"] = torch.empty(n, kh, d, dtype=TORCH[case["dst"]], device="cuda")
        weights()
    elif case["op"] == "append":
        lens, hist = _ints(case["lens"]), _ints(case["hist"])
        n = sum(lens)
        s["qkv"] = rand(n, h + 2 * kh, d, kind=case["src"])
        s["q"], s["k"], s["v"] = s["qkv"][:, :h], s["qkv"][:, h:h + kh], s["qkv"][:, h + kh:]
        s["q_out"] = torch.empty(n, h, d, dtype=TORCH[case["src"]], device="cuda")
        s["kc"], s["vc"], s["table"] = _cache(case, g, [a + b for a, b in zip(lens, hist)])
        s["seq"] = _dev([i for i, a in enumerate(lens) for _ in range(a)])
        s["pos"] = _dev([b + j for a, b in zip(lens, hist) for j in range(a)])
        weights()
    elif case["op"] == "prompt":
        lens, hist = _ints(case["lens"]), _ints(case["hist"])
        s["q"] = rand(sum(lens), h, d, kind=case["q"])
        s["out"] = torch.empty_like(s["q"])
        s["kc"], s["vc"], s["table"] = _cache(case, g, [a + b for a, b in zip(lens, hist)])
        s["cu"] = _dev([sum(lens[:i]) for i in range(len(lens) + 1)])
        s["kv_len"] = _dev([a + b for a, b in zip(lens, hist)])
        s["max_q"], s["max_kv"] = max(lens), max(a + b for a, b in zip(lens, hist))
    else:
        lens = _ints(case["lens"])
        s["q"] = rand(len(lens), h, d, kind=case["q"])
        s["out"] = torch.empty_like(s["q"])
        s["kc"], s["vc"], both = _cache(case, g, lens + [case["prefix"]])
        s["table"], s["prefix_table"] = both[:-1], both[-1]
        s["kv_len"] = _dev(lens)
        s["max_kv"] = max(lens)
    return s


# ----------------------------------------------------------- the plain form

def _thetas(case, device):
    """Angles per position of the rotating pairs (fp64), and the magnitude."""
    rot = case["rot"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    theta = torch.exp(i * (-2.0 * math.log(BASE) / rot))
    if case["scaling"] == "linear":
        return theta / case["factor"], 1.0
    if case["scaling"] == "yarn":
        lo, hi = (rot * math.log(ORIG_CTX / (2 * math.pi * b)) / (2 * math.log(BASE)) for b in (BETA_FAST, BETA_SLOW))
        ramp = ((i - lo) / (hi - lo)).clamp(0, 1)
        return theta * ((1 - ramp) + ramp / case["factor"]), 1.0 + 0.1 * math.log(case["factor"])
    return theta, 1.0


def _rotated(case, x, w, pos):
    """Rows [tokens][heads][dim] normalised per head and rotated, in fp32."""
    x = x.float()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    theta, mag = _thetas(case, x.device)
    angle = pos.double()[:, None] * theta
    c = (torch.cos(angle) * mag).float()[:, None, :]
    s = (torch.sin(angle) * mag).float()[:, None, :]
    rot = case["rot"]
    y = x.clone()
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2] = a * c - b * s
        y[..., rot // 2:rot] = b * c + a * s
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = a * c - b * s
        y[..., 1:rot:2] = b * c + a * s
    return y


def _gather(cache, table, rows):
    """Rows 0..rows-1 of every sequence of the table, [sequences][kv heads][rows][dim] in fp32."""
    page = cache.shape[1]
    t = table[:, :(rows + page - 1) // page].long()
    x = cache[t].flatten(1, 2)[:, :rows]
    return x.permute(0, 2, 1, 3).float()


def _plain_prompt(s):
    case, cu = s["case"], s["cu"].long()
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    lq, lk = s["max_q"], s["max_kv"]
    n, total = cu.numel() - 1, s["q"].shape[0]
    k, v = _gather(s["kc"], s["table"], lk), _gather(s["vc"], s["table"], lk)
    row = (cu[:-1, None] + torch.arange(lq, device="cuda")).clamp(max=total - 1)
    q = s["q"][row].float().view(n, lq, kh, h // kh, d).permute(0, 2, 3, 1, 4).reshape(n, kh, -1, d)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).view(n, h, lq, lk)
    kv_len = s["kv_len"].long()
    at = (kv_len - (cu[1:] - cu[:-1]))[:, None] + torch.arange(lq, device="cuda")
    seen = torch.arange(lk, device="cuda") <= at[:, :, None]
    x.masked_fill_(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = x.sub_(top).exp_()
    o = torch.matmul(e.view(n, kh, -1, lk), v).view(n, h, lq, d) / e.sum(-1, keepdim=True)
    t = torch.arange(total, device="cuda")
    i = torch.searchsorted(cu, t, right=True) - 1
    return o[i, :, t - cu[i]].to(s["q"].dtype)


def _plain_decode(s):
    case = s["case"]
    h, kh, d, p = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
    n, lk = s["q"].shape[0], s["max_kv"]
    q = s["q"].float().view(n, kh, h // kh, d)
    k, v = _gather(s["kc"], s["table"], lk), _gather(s["vc"], s["table"], lk)
    x = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    x.masked_fill_((torch.arange(lk, device="cuda") >= s["kv_len"].long()[:, None])[:, None, None], -math.inf)
    if p == 0:
        e = x.sub_(x.amax(-1, keepdim=True)).exp_()
        return (torch.matmul(e, v) / e.sum(-1, keepdim=True)).reshape(n, h, d).to(s["q"].dtype)
    pk, pv = _gather(s["kc"], s["prefix_table"][None], p)[0], _gather(s["vc"], s["prefix_table"][None], p)[0]
    y = torch.matmul(q.transpose(0, 1).reshape(kh, -1, d), pk.transpose(-1, -2)) * d ** -0.5
    y = y.view(kh, n, h // kh, p).transpose(0, 1)
    top = torch.maximum(x.amax(-1, keepdim=True), y.amax(-1, keepdim=True))
    e, f = torch.exp(x - top), torch.exp(y - top)
    o = torch.matmul(f.transpose(0, 1).reshape(kh, -1, p), pv).view(kh, n, h // kh, d).transpose(0, 1)
    o = (o + torch.matmul(e, v)) / (e.sum(-1, keepdim=True) + f.sum(-1, keepdim=True))
    return o.reshape(n, h, d).to(s["q"].dtype)


def _plain(s):
    case = s["case"]
    if case["op"] == "rotary":
        dst = TORCH[case["dst"]]
        return (_rotated(case, s["q"], s["qw"], s["pos"]).to(dst), _rotated(case, s["k"], s["kw"], s["pos"]).to(dst))
    if case["op"] == "append":
        page = case["page"]
        pos = s["pos"].long()
        at = s["table"][s["seq"].long(), pos // page].long()
        s["kc"][at, pos % page] = _rotated(case, s["k"], s["kw"], s["pos"]).to(s["kc"].dtype)
        s["vc"][at, pos % page] = s["v"].to(s["vc"].dtype)
        return (_rotated(case, s["q"], s["qw"], s["pos"]).to(s["q"].dtype), s["kc"], s["vc"])
    return _plain_prompt(s) if case["op"] == "prompt" else _plain_decode(s)


# ------------------------------------------------------- the library's calls

def _rows(t):
    from tensoros_b200 import _ffi
    return _ffi.Rows(t.data_ptr(), t.stride(0), F32 if t.dtype == torch.float32 else F16)


def _bound(s):
    """The descriptors and the workspace that a user's program keeps for this
    shape, and the call made of them."""
    import ctypes as C

    from tensoros_b200 import _ffi, lib
    case, L = s["case"], lib()
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    keep = []

    def ref(x):
        keep.append(x)
        return C.byref(x)

    def ptr(t):
        return None if t is None else t.data_ptr()

    if "kc" in s:
        kv = ref(_ffi.PagedKv(s["kc"].data_ptr(), s["vc"].data_ptr(), CODE[case["kv"]], s["kc"].shape[0],
                              case["page"], kh, d, s["table"].data_ptr(), s["table"].shape[0], s["table"].stride(0)))
    if case["op"] in ("rotary", "append"):
        desc = _ffi.RotaryDesc(rot_dim=case["rot"], layout=int(case["layout"] == "half"), base=BASE,
                               scaling=["none", "linear", "yarn"].index(case["scaling"]), factor=case["factor"],
                               orig_ctx=ORIG_CTX, beta_fast=BETA_FAST, beta_slow=BETA_SLOW, attn_factor=1.0,
                               freq_factors=None)
        plan = C.c_void_p()
        if L.tos_rotary_create(C.byref(plan), C.byref(desc)):
            raise RuntimeError("tos_rotary_create failed")
        q, k, q_out = ref(_rows(s["q"])), ref(_rows(s["k"])), ref(_rows(s["q_out"]))
    if case["op"] == "rotary":
        args = (q, q_out, k, ref(_rows(s["k_out"])), case["tokens"], h, kh, d, ptr(s["qw"]), ptr(s["kw"]), EPS, plan,
                s["pos"].data_ptr())
        return L.tos_qk_norm_rotary_dev, args, (s["q_out"], s["k_out"]), keep
    if case["op"] == "append":
        args = (kv, k, ref(_rows(s["v"])), q, q_out, s["q"].shape[0], h, s["seq"].data_ptr(), s["pos"].data_ptr(),
                s["pos"].data_ptr(), ptr(s["qw"]), ptr(s["kw"]), EPS, plan)
        return L.tos_kv_append_paged_dev, args, (s["q_out"], s["kc"], s["vc"]), keep
    q, out, total = ref(_rows(s["q"])), ref(_rows(s["out"])), s["q"].shape[0]
    if case["op"] == "prompt":
        n = L.tos_attention_prompt_paged_workspace_bytes(s["kv_len"].numel(), total, s["max_q"], s["max_kv"], h, kh, d)
    else:
        n = L.tos_attention_decode_paged_workspace_bytes(total, s["max_kv"], case["prefix"], h, kh, d)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device="cuda")
    keep.append(ws)
    if case["op"] == "prompt":
        args = (out, q, kv, s["cu"].data_ptr(), s["kv_len"].data_ptr(), s["kv_len"].numel(), total, s["max_q"],
                s["max_kv"], h, d ** -0.5, ws.data_ptr(), n)
        return L.tos_attention_prompt_paged_dev, args, s["out"], keep
    args = (out, q, kv, s["kv_len"].data_ptr(), total, s["max_kv"], s["prefix_table"].data_ptr(), case["prefix"], h,
            d ** -0.5, ws.data_ptr(), n)
    return L.tos_attention_decode_paged_dev, args, s["out"], keep


def run(s):
    if not own:
        return _plain(s)
    if "call" not in s:
        s["call"] = _bound(s)
    entry, args, out, _ = s["call"]
    # the library takes a null stream as its own; 1 is CUDA's legacy default stream
    status = entry(*args, torch.cuda.current_stream().cuda_stream or 1)
    if status:
        raise RuntimeError("%s: status %d" % (s["case"]["op"], status))
    return out


# ---------------------------------------------------- the definition in fp64

def _exact_heads(case, x, w, pos):
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    rot, out = case["rot"], x.clone()
    half = rot // 2
    for i in range(half):
        f, mag = BASE ** (-2.0 * i / rot), 1.0
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "yarn":
            edge = [rot * math.log(ORIG_CTX / (b * 2 * math.pi)) / (2 * math.log(BASE)) for b in (BETA_FAST, BETA_SLOW)]
            r = min(1.0, max(0.0, (i - edge[0]) / (edge[1] - edge[0])))
            f = r * f / case["factor"] + (1.0 - r) * f
            mag = 0.1 * math.log(case["factor"]) + 1.0
        z = torch.polar(torch.full_like(pos, mag, dtype=torch.float64), pos.double() * f)
        a, b = (i, i + half) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        y = torch.complex(x[..., a], x[..., b]) * z[:, None]
        out[..., a], out[..., b] = y.real, y.imag
    return out


def _exact_rows(cache, table_row, n):
    page = cache.shape[1]
    j = torch.arange(n, device="cuda")
    return cache[table_row.long()[j // page], j % page].double()     # [n][kv heads][dim]


def _exact_attend(q, k, v, scale, last):
    """q [rows][dim], k and v [keys][dim] in fp64; row r sees keys 0..last[r]."""
    x = (q @ k.T) * scale
    x = torch.where(torch.arange(k.shape[0], device="cuda")[None] <= last[:, None], x, -math.inf)
    return torch.softmax(x, -1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return (_exact_heads(case, s["q"], s["qw"], s["pos"]), _exact_heads(case, s["k"], s["kw"], s["pos"]))
    if case["op"] == "append":
        kc, vc = s["kc"].double(), s["vc"].double()
        page = case["page"]
        where = s["table"][s["seq"].long(), (s["pos"] // page).long()].long() * page + (s["pos"] % page).long()
        kc.view(-1, *kc.shape[2:])[where] = _exact_heads(case, s["k"], s["kw"], s["pos"])
        vc.view(-1, *vc.shape[2:])[where] = s["v"].double()
        return (_exact_heads(case, s["q"], s["qw"], s["pos"]), kc, vc)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "prompt":
        at = 0
        for i, (n, b) in enumerate(zip(_ints(case["lens"]), _ints(case["hist"]))):
            k, v = _exact_rows(s["kc"], s["table"][i], n + b), _exact_rows(s["vc"], s["table"][i], n + b)
            last = b + torch.arange(n, device="cuda")
            for j in range(h):
                out[at:at + n, j] = _exact_attend(s["q"][at:at + n, j].double(), k[:, j * kh // h], v[:, j * kh // h],
                                                  d ** -0.5, last)
            at += n
        return out
    p = case["prefix"]
    pk, pv = _exact_rows(s["kc"], s["prefix_table"], p), _exact_rows(s["vc"], s["prefix_table"], p)
    for i, n in enumerate(_ints(case["lens"])):
        k = torch.cat([pk, _exact_rows(s["kc"], s["table"][i], n)])
        v = torch.cat([pv, _exact_rows(s["vc"], s["table"][i], n)])
        for j in range(kh):
            rows = slice(j * (h // kh), (j + 1) * (h // kh))
            out[i, rows] = _exact_attend(s["q"][i, rows].double(), k[:, j], v[:, j], d ** -0.5,
                                         torch.full((h // kh,), p + n, device="cuda"))
    return out
