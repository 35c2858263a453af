"""What a batch of sequences needs around its paged cache, as cases to time and compare.

Four operators of include/krafla_hip.h and what they compute, written out in
elementary torch operations (own = False):

  share   krh_paged_attention_shared: one new token of each sequence, the first
          rows of a group of sequences read once for the group
  i8      krh_matmul_i8: products of 8-bit integers, a scale a token and a
          scale an output
  glu     krh_matmul_i8_swiglu: the two products of a gated FFN and its
          activation
  norm    krh_block_norm: the norm after a block, its gate, the residual add and
          the next block's norm, as floats or as 8-bit rows (which
          krh_dequantize_row_rows gives back as the values that they stand for)

Sizes are those of the repository's own configurations (stories15M, the 0.5B,
1B and 8B shapes, Gemma-like heads) or generic ones.
"""
import ctypes as C
import math
import os
import random
import sys

import torch

own = False

EPS = 2.0 ** -20   # the same in 32 bits and in 64
HEADS = {"15m": (6, 6, 48), "0.5b": (14, 2, 64), "1b": (32, 8, 64), "8b": (32, 8, 128), "gemma": (8, 4, 256)}
WIDTH = {"f32": 4, "f16": 2, "q8": 1}
# the largest cases: query times key values, the pool's bytes, a product's operations, a norm's values
SHARE_MOST = 64 * 32 * 128 * 34000
POOL_MOST = 1 << 30
I8_MOST = 2047 * 4096 * 14336
NORM_MOST = 2047 * 4096


def _heads(shape):
    nh, nkv, hd = HEADS[shape]
    return dict(heads=nh, kv_heads=nkv, head_dim=hd)


def listed():
    return [
        # a few users of one short system prompt: latency alone
        dict(name="share_05b_few", kind="share", **_heads("0.5b"), kv="f16", page=16, seqs=4, groups=1, shared=208,
             rows=90, window=0, softcap=0.0),
        # a batch of chats behind one instruction, 8B shape
        dict(name="share_8b_batch", kind="share", **_heads("8b"), kv="f16", page=16, seqs=16, groups=1, shared=2048,
             rows=1001, window=0, softcap=0.0),
        # a full server: 64 questions about one long document, 8B shape
        dict(name="share_8b_server", kind="share", **_heads("8b"), kv="f16", page=64, seqs=64, groups=1, shared=32000,
             rows=2000, window=0, softcap=0.0),
        # an 8-bit cache, three assistants with a prompt each, 1B shape
        dict(name="share_1b_q8", kind="share", **_heads("1b"), kv="q8", page=32, seqs=48, groups=3, shared=6016,
             rows=700, window=0, softcap=0.0),
        # a sliding-window layer with capped scores over a float cache: of the prompt its end is attended
        dict(name="share_gemma_window", kind="share", **_heads("gemma"), kv="f32", page=16, seqs=8, groups=1,
             shared=1504, rows=600, window=1024, softcap=50.0),
        # one token of the 15M shape, its FFN's first product
        dict(name="i8_15m_token", kind="i8", tokens=1, rows=768, cols=288, bias=False, add=False),
        # a step of 16 sequences: the 8B shape's FFN output into the residual
        dict(name="i8_8b_step", kind="i8", tokens=16, rows=4096, cols=14336, bias=False, add=True),
        # a prompt's attention projection with its bias, 8B shape
        dict(name="i8_8b_prompt", kind="i8", tokens=2047, rows=4096, cols=4096, bias=True, add=False),
        # a step of a hundred sequences, 1B shape
        dict(name="glu_1b_batch", kind="glu", tokens=100, rows=8192, cols=2048),
        # a prompt, 8B shape
        dict(name="glu_8b_prompt", kind="glu", tokens=2047, rows=14336, cols=4096),
        # between two blocks of a step of 16 sequences, 8B shape
        dict(name="norm_8b_step", kind="norm", tokens=16, n=4096, post=True, gate="none", out="z"),
        # between two blocks of a prompt, into the 8-bit product that follows
        dict(name="norm_8b_prompt", kind="norm", tokens=2047, n=4096, post=True, gate="channel", out="q"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["share", "share", "i8", "i8", "glu", "norm"])
    if kind == "norm":
        n = _log(rng, 8, 16384)
        return dict(kind=kind, tokens=_log(rng, 1, min(2047, NORM_MOST // n)), n=n, post=rng.random() < 0.5,
                    gate=rng.choice(["none", "channel", "token"]), out=rng.choice(["z", "q", "zq", "none"]))
    if kind in ("i8", "glu"):
        rows, cols = _log(rng, 16, 14336), _log(rng, 16, 14336)
        most = (2 if kind == "glu" else 4) * I8_MOST // 2
        s = dict(kind=kind, tokens=_log(rng, 1, min(2047, most // (rows * cols))), rows=rows, cols=cols)
        return dict(s, bias=rng.random() < 0.5, add=rng.random() < 0.5) if kind == "i8" else s
    nkv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([48, 64, 64, 80, 96, 128, 128, 256])
    s = dict(kind=kind, heads=nkv * rng.choice([1, 2, 3, 4, 7, 8, 16]), kv_heads=nkv, head_dim=hd,
             kv=rng.choice(["f32", "f16", "f16", "q8"]), page=rng.choice([16, 16, 32, 64, 128, 256]))
    row = 2 * nkv * hd * WIDTH[s["kv"]]
    seqs = _log(rng, 1, 64)
    groups = rng.randrange(1, min(4, seqs) + 1)
    both = SHARE_MOST // (seqs * s["heads"] * hd)
    shared = _log(rng, 16, max(17, min(32000, both, POOL_MOST // row // groups)))
    # the plain form holds own rows in 32 bits
    own_rows = _log(rng, 1, max(2, min(4000, both - shared, POOL_MOST // row // seqs, (3 << 30) // (4 * seqs * nkv * hd))))
    return dict(s, seqs=seqs, groups=groups, shared=shared // s["page"] * s["page"], rows=own_rows,
                window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]))


# ---- how a batch is made up: numbers of the case alone ----

def _own_rows(case):
    """rows of each sequence behind the shared ones: one the most, the others of all lengths"""
    rng = random.Random(case["seqs"] * 1009 + case["rows"])
    return [case["rows"]] + [_log(rng, 1, case["rows"]) for _ in range(case["seqs"] - 1)]


def _groups(case):
    """(first sequence, sequences, shared rows) of each group: the first's prompt the longest"""
    rng = random.Random(case["seqs"] * 31 + case["shared"])
    cut = [0] + sorted(rng.sample(range(1, case["seqs"]), case["groups"] - 1)) + [case["seqs"]]
    p = case["page"]
    shared = [case["shared"]] + [_log(rng, max(1, case["shared"] // 4), max(1, case["shared"])) // p * p
                                 for _ in range(case["groups"] - 1)]
    return [(a, b - a, n) for a, b, n in zip(cut, cut[1:], shared)]


# ---- inputs ----

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _q8(x):
    """int8 rows of one scale each, the quotients rounded once from 64 bits"""
    m = x.abs().amax(-1, keepdim=True)
    f = (127 / m.double()).float()
    q = torch.trunc(x * f + torch.copysign(torch.full_like(x, 0.5), x)).clamp(-127, 127)
    zero = m < 1e-30
    return q.masked_fill(zero, 0.0), (m.double() / 127).float().masked_fill(zero, 0.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    s = dict(case)
    {"share": _prepare_share, "i8": _prepare_i8, "glu": _prepare_i8, "norm": _prepare_norm}[case["kind"]](s, g)
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_share(s, g):
    page = s["page"]
    rows, s["parts"] = _own_rows(s), _groups(s)
    lens = []
    for first, n, shared in s["parts"]:
        lens += [shared + rows[i] for i in range(first, first + n)]
    used = [-(-n // page) for n in lens]
    fresh = sum(sh // page for _, _, sh in s["parts"]) + sum(
        used[i] - sh // page for f, n, sh in s["parts"] for i in range(f, f + n))
    ids = torch.randperm(fresh, generator=g, device="cuda").int()
    table = torch.full((s["seqs"], max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for first, n, shared in s["parts"]:
        k = shared // page
        table[first:first + n, :k] = ids[at:at + k]
        at += k
        for i in range(first, first + n):
            table[i, k:used[i]] = ids[at:at + used[i] - k]
            at += used[i] - k
    s["table"], s["len"], s["most"] = table, _ints(lens), max(lens)
    s["start"] = _ints([f for f, _, _ in s["parts"]] + [s["seqs"]])
    s["prefix"] = _ints([sh for _, _, sh in s["parts"]])
    shape = (fresh, s["kv_heads"], page, s["head_dim"])
    p = s["pool"] = {}
    for n in ("k", "v"):
        if s["kv"] == "q8":
            p[n] = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda")
            p[n + "d"] = 0.012 + 0.012 * torch.rand(shape[:3], generator=g, device="cuda")
        else:
            p[n] = torch.empty(shape, dtype=torch.float16 if s["kv"] == "f16" else torch.float32,
                               device="cuda").normal_(generator=g)
    s["q"] = _randn(g, s["seqs"], s["heads"], s["head_dim"]) * 1.5


def _matrix(g, rows, cols):
    """an int8 matrix with a scale a row, as a caller keeps it: rows 16 bytes' multiples apart"""
    ld = -(-cols // 16) * 16
    q, d = _q8(_randn(g, rows, cols) * 0.02)
    w = torch.zeros(rows, ld, dtype=torch.int8, device="cuda")
    w[:, :cols] = q
    return w, d.view(-1).contiguous()


def _prepare_i8(s, g):
    s["w"] = [_matrix(g, s["rows"], s["cols"]) for _ in range(2 if s["kind"] == "glu" else 1)]
    # tokens of different sizes, a few channels far larger than the others, as a norm's outputs are
    x = _randn(g, s["tokens"], s["cols"]) * torch.exp(_randn(g, s["tokens"], 1))
    x[:, ::97] *= 8
    ld = -(-s["cols"] // 16) * 16
    q, d = _q8(x)
    s["xq"] = torch.zeros(s["tokens"], ld, dtype=torch.int8, device="cuda")
    s["xq"][:, :s["cols"]] = q
    s["xd"] = d.view(-1).contiguous()
    if s["kind"] == "i8":
        s["b"] = _randn(g, s["rows"]) if s["bias"] else None
        s["y0"] = _randn(g, s["tokens"], s["rows"]) if s["add"] else None


def _prepare_norm(s, g):
    t, n = s["tokens"], s["n"]
    s["x"] = _randn(g, t, n) * torch.exp(_randn(g, t, 1))
    s["y"] = _randn(g, t, n) * 0.3
    s["post_w"] = 1 + 0.1 * _randn(g, n) if s["post"] else None
    s["g"] = {"none": None, "channel": 0.5 + 0.2 * _randn(g, n), "token": torch.tanh(_randn(g, t, n))}[s["gate"]]
    s["alpha"] = 1.0 if s["gate"] == "none" else 0.70710678
    s["pre_w"] = 1 + 0.1 * _randn(g, n) if s["out"] != "none" else None


# ---- the framework's calls ----

def _binding():
    sys.path.insert(0, os.path.join(os.getcwd(), "isa-lm_amd"))   # run from the repository's root
    import krafla
    return krafla


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _prepare_own(s):
    K = _binding()
    K.init_device()
    h, dev = K.hip, dict(device="cuda", dtype=torch.float32)
    if s["kind"] == "share":
        p = s["pool"]
        s["pages"] = K.KrhPages(p["k"].data_ptr(), p["v"].data_ptr(), _ptr(p.get("kd")), _ptr(p.get("vd")),
                                {"f32": K.ML_F32, "f16": K.ML_F16, "q8": K.ML_Q8_0}[s["kv"]], p["k"].shape[0],
                                s["page"], s["kv_heads"], s["head_dim"])
        s["o"] = torch.empty_like(s["q"])
        n = h.krh_paged_attention_shared_ws(C.byref(s["pages"]), s["seqs"], s["heads"], s["most"], s["groups"],
                                            s["shared"])
        s["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    elif s["kind"] == "norm":
        t, n = s["tokens"], s["n"]
        s["xo"] = torch.empty(t, n, **dev)
        s["z"] = torch.empty(t, n, **dev) if "z" in s["out"] else None
        s["qo"] = torch.empty(t, -(-n // 16) * 16, dtype=torch.int8, device="cuda") if "q" in s["out"] else None
        s["d"] = torch.empty(t, 1, **dev) if "q" in s["out"] else None
        s["qv"] = torch.empty(t, n, **dev) if "q" in s["out"] else None
    else:
        s["mats"] = [K.KrhMat8(q.data_ptr(), d.data_ptr(), q.shape[1], s["rows"], s["cols"]) for q, d in s["w"]]
        s["yo"] = torch.empty(s["tokens"], s["rows"], **dev)


def _run_own(s):
    h = sys.modules["krafla"].hip
    if s["kind"] == "share":
        h.krh_paged_attention_shared(s["o"].data_ptr(), C.byref(s["pages"]), s["table"].data_ptr(), s["table"].shape[1],
                                     s["len"].data_ptr(), s["seqs"], s["start"].data_ptr(), s["prefix"].data_ptr(),
                                     s["groups"], s["shared"], s["q"].data_ptr(), s["heads"], s["most"], s["window"],
                                     s["head_dim"] ** -0.5, s["softcap"], s["ws"].data_ptr())
        return s["o"]
    if s["kind"] == "glu":
        h.krh_matmul_i8_swiglu(s["yo"].data_ptr(), s["rows"], C.byref(s["mats"][0]), C.byref(s["mats"][1]),
                               s["xq"].data_ptr(), s["xq"].shape[1], s["xd"].data_ptr(), s["tokens"])
        return s["yo"]
    if s["kind"] == "i8":
        if s["add"]:
            h.krh_copy_d2d_async(s["yo"].data_ptr(), s["y0"].data_ptr(), s["y0"].nbytes)
        h.krh_matmul_i8(s["yo"].data_ptr(), s["rows"], C.byref(s["mats"][0]), s["xq"].data_ptr(), s["xq"].shape[1],
                        s["xd"].data_ptr(), _ptr(s["b"]), s["tokens"], int(s["add"]))
        return s["yo"]
    n = s["n"]
    h.krh_block_norm(s["xo"].data_ptr(), n, s["x"].data_ptr(), n, s["y"].data_ptr(), n, _ptr(s["post_w"]), _ptr(s["g"]),
                     n if s["gate"] == "token" else 0, s["alpha"], _ptr(s["pre_w"]), EPS, _ptr(s["z"]), n,
                     _ptr(s["qo"]), s["qo"].shape[1] if s["qo"] is not None else 0, _ptr(s["d"]), n, s["tokens"])
    out = {"x": s["xo"]}
    if s["z"] is not None:
        out["z"] = s["z"]
    if s["qo"] is not None:
        h.krh_dequantize_row_rows(s["qv"].data_ptr(), n, s["qo"].data_ptr(), s["qo"].shape[1], s["d"].data_ptr(), 1, n,
                                  s["tokens"])
        out["q"] = s["qv"]
    return out


# ---- the plain forms ----

def run(s):
    if own:
        return _run_own(s)
    return {"share": _share, "i8": _i8, "glu": _glu, "norm": _norm}[s["kind"]](s)


def _rows(s, name, table, n):
    """[kv head][row][dim] of the first n rows of a table's pages (or [seq] of such) in 32 bits"""
    t = table.clamp(min=0).long()
    x = s["pool"][name][t].float()
    if name + "d" in s["pool"]:
        x = x * s["pool"][name + "d"][t].unsqueeze(-1)
    x = x.transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1])[..., :n, :].contiguous()


def _share(s):
    nkv, hd, page, most = s["kv_heads"], s["head_dim"], s["page"], max(s["rows"], 1)
    out = torch.empty_like(s["q"])
    for first, n, shared in s["parts"]:
        at = slice(first, first + n)
        q = s["q"][at].view(n, nkv, -1, hd)
        ln = s["len"][at].view(n, 1, 1, 1)
        # own rows a sequence, the shared ones of all sequences at once
        own_table = s["table"][at, shared // page:]
        k, v = (_rows(s, m, own_table, most) for m in ("k", "v"))
        z = torch.matmul(q, k.transpose(2, 3).contiguous())                       # [seq][kv head][head][row]
        if shared:
            k1, v1 = (_rows(s, m, s["table"][first, :shared // page], shared) for m in ("k", "v"))
            qs = q.transpose(0, 1).reshape(nkv, -1, hd)
            z1 = torch.matmul(qs, k1.transpose(1, 2).contiguous()).view(nkv, n, -1, shared).transpose(0, 1)
            z = torch.cat([z1, z], 3)
        z = z * hd ** -0.5
        if s["softcap"] > 0:
            z = s["softcap"] * torch.tanh(z / s["softcap"])
        row = torch.arange(z.shape[3], device="cuda")
        ok = row < ln
        if s["window"]:
            ok = ok & (row >= ln - s["window"])
        z = z.masked_fill(~ok, -math.inf)
        e = torch.exp(z - z.amax(3, keepdim=True))
        a = e / e.sum(3, keepdim=True)
        o = torch.matmul(a[..., shared:].contiguous(), v)
        if shared:
            a1 = a[..., :shared].transpose(0, 1).reshape(nkv, -1, shared)
            o = o + torch.matmul(a1, v1).view(nkv, n, -1, hd).transpose(0, 1)
        out[at] = o.reshape(n, -1, hd)
    return out


def _sums(s, i):
    """whole numbers: partial sums of 1024 products are exact in 32-bit floats"""
    x, w, c = s["xq"], s["w"][i][0], s["cols"]
    acc = torch.zeros(s["tokens"], s["rows"], dtype=torch.int32, device="cuda")
    for k in range(0, c, 1024):
        e = min(c, k + 1024)
        acc += torch.matmul(x[:, k:e].float(), w[:, k:e].float().t()).int()
    return acc.float() * s["xd"].unsqueeze(1) * s["w"][i][1]


def _i8(s):
    y = _sums(s, 0)
    if s["bias"]:
        y = y + s["b"]
    return s["y0"] + y if s["add"] else y


def _glu(s):
    g, u = _sums(s, 0), _sums(s, 1)
    return g / (1 + torch.exp(-g)) * u


def _inv(x):
    # the sum in 64 bits, so that an 8-bit value next to a border falls on one side of it
    return (1 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()


def _norm(s):
    y = s["y"]
    if s["post"]:
        y = y * _inv(y) * s["post_w"]
    if s["g"] is not None:
        y = y * s["g"]
    x = s["x"] + y * s["alpha"]
    out = {"x": x}
    if s["out"] != "none":
        z = x * _inv(x) * s["pre_w"]
        if "z" in s["out"]:
            out["z"] = z
        if "q" in s["out"]:
            q, d = _q8(z)
            out["q"] = q * d
    return out


# ---- what a pass cannot do without ----

def work(case):
    if case["kind"] == "norm":
        t, n = case["tokens"], case["n"]
        each = 12 + 4 * (case["gate"] == "token") + 4 * ("z" in case["out"])
        each += 6 if "q" in case["out"] else 0   # 8-bit values come back as what they stand for
        return dict(bytes=t * n * each, flops=12 * t * n)
    if case["kind"] in ("i8", "glu"):
        t, r, c, m = case["tokens"], case["rows"], case["cols"], 2 if case["kind"] == "glu" else 1
        out = 4 * t * r * (2 if case.get("add") else 1)
        return dict(bytes=m * r * (c + 4) + t * (c + 4) + out, flops=2 * m * t * r * c)
    hd, nh, nkv = case["head_dim"], case["heads"], case["kv_heads"]
    row = nkv * (2 * hd * WIDTH[case["kv"]] + (8 if case["kv"] == "q8" else 0))
    w = case["window"]
    rows, read, pairs = _own_rows(case), 0, 0
    for first, n, shared in _groups(case):
        lens = [shared + rows[i] for i in range(first, first + n)]
        seen = [min(v, w) if w else v for v in lens]
        read += sum(min(a, v - shared) for a, v in zip(seen, lens))
        read += max(0, shared - min(v - a for v, a in zip(lens, seen)))
        pairs += sum(seen)
    return dict(bytes=read * row + 8 * case["seqs"] * nh * hd, flops=4 * nh * hd * pairs)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"share": _share_exact, "i8": _i8_exact, "glu": _i8_exact, "norm": _norm_exact}[case["kind"]](s)


def _share_exact(s):
    nkv, hd = s["kv_heads"], s["head_dim"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["len"].tolist()):
        at = torch.arange(max(0, n - s["window"]) if s["window"] else 0, n, device="cuda")
        page, slot = s["table"][i].long()[at // s["page"]], at % s["page"]
        k, v = (s["pool"][m][page, :, slot].double() for m in ("k", "v"))
        if s["kv"] == "q8":
            k, v = (x * s["pool"][m + "d"][page, :, slot].double().unsqueeze(-1) for x, m in ((k, "k"), (v, "v")))
        for g in range(nkv):
            h = slice(g * s["heads"] // nkv, (g + 1) * s["heads"] // nkv)
            z = s["q"][i, h].double() @ k[:, g].t().contiguous() / math.sqrt(hd)
            if s["softcap"] > 0:
                z = s["softcap"] * torch.tanh(z / s["softcap"])
            o[i, h] = torch.softmax(z, 1) @ v[:, g].contiguous()
    return o


def _i8_exact(s):
    x = s["xq"][:, :s["cols"]].double()
    y = [x @ q[:, :s["cols"]].double().t().contiguous() * s["xd"].double()[:, None] * d.double()[None] for q, d in s["w"]]
    if s["kind"] == "glu":
        return torch.nn.functional.silu(y[0]) * y[1]
    y = y[0]
    if s["b"] is not None:
        y += s["b"].double()
    return y + s["y0"].double() if s["y0"] is not None else y


def _norm_exact(s):
    def scaled(v, w):
        return v / torch.sqrt((v * v).sum(1, keepdim=True) / s["n"] + EPS) * w.double()

    y = s["y"].double()
    if s["post_w"] is not None:
        y = scaled(y, s["post_w"])
    if s["g"] is not None:
        y = y * s["g"].double()
    x = s["x"].double() + s["alpha"] * y
    out = {"x": x}
    if "z" in s["out"]:
        out["z"] = scaled(x, s["pre_w"])
    if "q" in s["out"]:
        # which of two 8-bit values holds is decided by the rule's 32-bit
        # products, so what they stand for has no other form in 64 bits
        out["q"] = None
    return out


if __name__ == "__main__":
    for number in range(6):
        print(draw(random.Random(number)))
