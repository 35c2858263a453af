"""The decode step of several sequences over a paged cache, as cases to time and compare.

Four operators of include/krafla_hip.h and what they compute, written out in
elementary torch operations (own = False):

  qkv     krh_paged_qkv: query and key heads normalized and rotated at each
          row's own position, K and V into their pages
  attn    krh_paged_attention: one new token of each sequence over its pages
  evict   krh_paged_evict: the heaviest and the latest rows of each KV head
          into other pages
  rules   krh_logit_rules: penalties, biases and token masks on logit rows

Sizes are those of the repository's own configurations (stories15M, the 0.5B,
1B and 8B shapes, Gemma-like heads) or generic ones. Row r of a sequence lies in
page table[r // page], slot r % page; a page holds [kv head][slot][dim].
"""
import ctypes as C
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
HEADS = {"15m": (6, 6, 48), "0.5b": (14, 2, 64), "1b": (32, 8, 64), "8b": (32, 8, 128), "gemma": (8, 4, 256)}
WIDTH = {"f32": 4, "f16": 2, "q8": 1}
ROWS_MOST = 64 * 6144 * 8 * 128 * 4   # bytes of K and V in the largest case


def _heads(shape):
    nh, nkv, hd = HEADS[shape]
    return dict(heads=nh, kv_heads=nkv, head_dim=hd)


def listed():
    return [
        # the first tokens after a short prompt, one user: latency alone
        dict(name="attn_05b_short", kind="attn", **_heads("0.5b"), kv="f16", page=16, seqs=1, rows=37, window=0,
             softcap=0.0, mass=False),
        # a batch of chats of all lengths, 8B shape
        dict(name="attn_8b_batch", kind="attn", **_heads("8b"), kv="f16", page=16, seqs=16, rows=4001, window=0,
             softcap=0.0, mass=False),
        # one long document, 8B shape: few rows, a long axis
        dict(name="attn_8b_long", kind="attn", **_heads("8b"), kv="f16", page=64, seqs=1, rows=120001, window=0,
             softcap=0.0, mass=False),
        # an 8-bit cache whose weights are accumulated for its eviction, 1B shape
        dict(name="attn_1b_q8_mass", kind="attn", **_heads("1b"), kv="q8", page=32, seqs=24, rows=8100, window=0,
             softcap=0.0, mass=True),
        # a sliding-window layer with capped scores over a float cache
        dict(name="attn_gemma_window", kind="attn", **_heads("gemma"), kv="f32", page=16, seqs=8, rows=2500,
             window=1024, softcap=50.0, mass=False),
        # a full server: 64 sequences, 8B shape
        dict(name="attn_8b_server", kind="attn", **_heads("8b"), kv="f16", page=64, seqs=64, rows=6144, window=0,
             softcap=0.0, mass=False),
        # the new token of 16 sequences, each at its own position
        dict(name="qkv_8b_step", kind="qkv", **_heads("8b"), kv="f16", page=16, seqs=16, tokens=16, norm=False),
        # two prompts at once into an 8-bit cache, heads normalized
        dict(name="qkv_1b_prompt", kind="qkv", **_heads("1b"), kv="q8", page=32, seqs=2, tokens=2047, norm=True),
        # 16 long chats cut to half their budget
        dict(name="evict_8b_batch", kind="evict", **_heads("8b"), kv="f16", page=16, seqs=16, rows=4096, keep=2048,
             recent=512),
        # one long document's 8-bit cache cut to an eighth
        dict(name="evict_1b_long", kind="evict", **_heads("1b"), kv="q8", page=32, seqs=1, rows=32001, keep=4000,
             recent=250),
        # one user's step of the 15M model
        dict(name="rules_one", kind="rules", vocab=32000, rows=1, seen=70, biases=5, masks=1),
        # a batch over the largest vocabulary, half of the rows under a grammar
        dict(name="rules_batch", kind="rules", vocab=151936, rows=64, seen=2000, biases=300, masks=32),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "qkv", "evict", "rules"])
    if kind == "rules":
        return dict(kind=kind, vocab=_log(rng, 500, 151936), rows=_log(rng, 1, 64), seen=_log(rng, 1, 8000),
                    biases=rng.choice([0, _log(rng, 1, 1000)]), masks=rng.choice([0, _log(rng, 1, 64)]))
    nkv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([48, 64, 64, 80, 96, 128, 128, 256])
    s = dict(kind=kind, heads=nkv * rng.choice([1, 2, 3, 4, 7, 8, 16]), kv_heads=nkv, head_dim=hd,
             kv=rng.choice(["f32", "f16", "f16", "q8"]), page=rng.choice([16, 16, 32, 64, 128, 256]))
    row = 2 * nkv * hd * WIDTH[s["kv"]]
    if kind == "qkv":
        tokens = _log(rng, 1, 2047)
        return dict(s, seqs=rng.randrange(1, min(64, tokens) + 1), tokens=tokens, norm=rng.random() < 0.5)
    seqs = _log(rng, 1, 64)
    if kind == "evict":
        rows = _log(rng, 40, max(41, min(32000, ROWS_MOST // 16 // row // seqs)))
        keep = rng.randrange(1, rows)
        return dict(s, seqs=seqs, rows=rows, keep=keep, recent=rng.randrange(0, keep + 1))
    rows = _log(rng, 1, min(120001, ROWS_MOST // row // seqs))
    # the plain form holds a score a head and row, and K and V in 32 bits
    rows = max(1, min(rows, (3 << 30) // (4 * seqs * max(s["heads"] * 4, nkv * hd))))
    return dict(s, seqs=seqs, rows=rows, window=rng.choice([0, 0, _log(rng, 16, 4096)]),
                softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), mass=rng.random() < 0.3)


def _lens(case, most):
    """Rows of each sequence: one the longest, the others of all lengths from a few on."""
    rng = random.Random(case["seqs"] * 1009 + most)
    return [most] + [_log(rng, max(1, most // 8), most) for _ in range(case["seqs"] - 1)]


# ---- inputs ----

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(g, case, pages, filled):
    """`pages` pages, the first `filled` of them with normal values (8 bits: with
    scales of a row's maximum over 127), the others zero."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    s = {}
    for n in ("k", "v"):
        if case["kv"] == "q8":
            s[n] = torch.zeros(shape, dtype=torch.int8, device="cuda")
            s[n + "d"] = torch.zeros(shape[:3], device="cuda")
            s[n][:filled] = torch.randint(-127, 128, (filled,) + shape[1:], generator=g, dtype=torch.int8, device="cuda")
            s[n + "d"][:filled] = 0.012 + 0.012 * torch.rand((filled,) + shape[1:3], generator=g, device="cuda")
        else:
            s[n] = torch.zeros(shape, dtype=torch.float16 if case["kv"] == "f16" else torch.float32, device="cuda")
            s[n][:filled].normal_(generator=g)
    return s


def _table(g, lens, page, first=0):
    """Each sequence's pages in no order, -1 behind them; and how many there are."""
    used = [-(-n // page) for n in lens]
    ids = (torch.randperm(sum(used), generator=g, device="cuda") + first).split(used)
    return torch.nn.utils.rnn.pad_sequence(ids, batch_first=True, padding_value=-1).int().contiguous(), sum(used)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    s = dict(case)
    if case["kind"] == "rules":
        _prepare_rules(s, g)
    else:
        {"attn": _prepare_attn, "qkv": _prepare_qkv, "evict": _prepare_evict}[case["kind"]](s, g)
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_attn(s, g):
    lens = _lens(s, s["rows"])
    s["table"], n = _table(g, lens, s["page"])
    s["pool"], s["len"] = _pool(g, s, n, n), _ints(lens)
    s["q"] = _randn(g, s["seqs"], s["heads"], s["head_dim"]) * 1.5
    s["mass0"] = _randn(g, s["seqs"], s["kv_heads"], s["rows"]).abs() if s["mass"] else None


def _prepare_qkv(s, g):
    # the tokens of a sequence are its next rows, at positions of their own (rows
    # have been evicted before them)
    T, n, hd = s["tokens"], s["seqs"], s["head_dim"]
    seq = torch.sort(torch.cat([torch.arange(n), torch.arange(T - n) % n]))[0]
    at = torch.arange(T) - torch.searchsorted(seq, seq)
    start = torch.arange(n) * 13 % 50
    s["seq"], s["row"] = seq.int().cuda(), (start[seq] + at).int().cuda()
    s["pos"] = (start[seq] * 40 + at).int().cuda()
    s["table"], pages = _table(g, [int(v) + int((seq == i).sum()) for i, v in enumerate(start)], s["page"])
    s["pool"] = _pool(g, s, pages, 0)
    s["q"] = _randn(g, T, s["heads"] * hd)
    s["k"], s["v"] = _randn(g, T, s["kv_heads"] * hd), _randn(g, T, s["kv_heads"] * hd)
    s["qw"], s["kw"] = (1 + 0.1 * _randn(g, hd) if s["norm"] else None for _ in range(2))
    ang = torch.arange(4096, dtype=torch.float64).unsqueeze(1) * 5e5 ** (-torch.arange(hd // 2).double() * 2 / hd)
    s["cos"], s["sin"] = ang.cos().float().cuda(), ang.sin().float().cuda()


def _prepare_evict(s, g):
    lens = _lens(s, s["rows"])
    kept = [min(n, s["keep"]) for n in lens]
    s["table"], n = _table(g, lens, s["page"])
    s["out_table"], m = _table(g, kept, s["page"], n)
    s["pool"], s["first"], s["len"] = _pool(g, s, n + m, n), n, _ints(lens)
    # weights as attention leaves them: most rows little, some much, and equal
    # ones (rows that no head looked at, or few times)
    w = _randn(g, s["seqs"], s["kv_heads"], s["rows"])
    s["weight"] = torch.where(w < -0.5, torch.zeros_like(w), torch.exp(2 * w))
    s["weight"] *= torch.arange(s["rows"], device="cuda") < s["len"].view(-1, 1, 1)
    s["lseq"] = torch.repeat_interleave(torch.arange(s["seqs"]), torch.tensor(kept)).int().cuda()
    s["lrow"] = torch.cat([torch.arange(n) for n in kept]).int().cuda()


def _prepare_rules(s, g):
    r, v = s["rows"], s["vocab"]
    s["logits"] = _randn(g, r, v) * 2.5
    # ids seen: common ones often, as text has them
    s["ids"] = (v ** torch.rand(r, s["seen"], generator=g, device="cuda") - 1).int().clamp(0, v - 1)
    s["n_ids"] = _ints([max(0, s["seen"] - 7 * i * s["seen"] // (8 * r)) for i in range(r)])
    s["repeat"] = 1 + 0.3 * torch.rand(r, generator=g, device="cuda")
    s["presence"], s["frequency"] = (0.5 * torch.rand(r, generator=g, device="cuda") for _ in range(2))
    b = max(1, s["biases"])
    s["bias_ids"] = torch.randint(0, v, (r, b), generator=g, dtype=torch.int32, device="cuda")
    s["bias_ids"][:, b // 2] = s["bias_ids"][:, 0]   # one id twice
    s["bias"] = _randn(g, r, b) * 3
    s["n_bias"] = _ints([s["biases"] if i % 3 else s["biases"] // 2 for i in range(r)])
    # masks of a few ids and of most ids in turn, on every other row
    m = max(1, s["masks"])
    share = torch.tensor([0.01, 0.97], device="cuda").repeat(m)[:m].view(-1, 1, 1)
    bits = torch.rand(m, (v + 31) // 32, 32, generator=g, device="cuda") < share
    s["bits"] = (bits.long() << torch.arange(32, device="cuda")).sum(2).to(torch.int32)
    s["mask"] = _ints([(i // 2) % m if s["masks"] and i % 2 == 0 else -1 for i in range(r)])


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
    if s["kind"] == "rules":
        row = torch.stack([s["repeat"], s["presence"], s["frequency"]], 1).view(torch.int32)
        s["rule"] = torch.cat([row, s["mask"].unsqueeze(1)], 1).contiguous()
        s["out"] = torch.empty_like(s["logits"])
        return
    p = s["pool"]
    s["pages"] = K.KrhPages(p["k"].data_ptr(), p["v"].data_ptr(), _ptr(p.get("kd")), _ptr(p.get("vd")),
                            {"f32": K.ML_F32, "f16": K.ML_F16, "q8": K.ML_Q8_0}[s["kv"]], p["k"].shape[0], s["page"],
                            s["kv_heads"], s["head_dim"])
    nkv, hd = s["kv_heads"], s["head_dim"]
    if s["kind"] == "attn":
        s["o"] = torch.empty(s["seqs"], s["heads"], hd, **dev)
        s["mass1"] = torch.empty_like(s["mass0"]) if s["mass"] else None
        n = h.krh_paged_attention_ws(C.byref(s["pages"]), s["seqs"], s["heads"], s["rows"], int(s["mass"]))
        s["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    elif s["kind"] == "qkv":
        s["qo"] = torch.empty_like(s["q"])
        n = s["tokens"]
    else:
        s["weight1"] = torch.empty(s["seqs"], nkv, s["keep"], **dev)
        s["len1"] = torch.empty_like(s["len"])
        n = h.krh_paged_evict_ws(s["seqs"], nkv, s["keep"])
        s["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        n = s["lseq"].numel()
    if s["kind"] != "attn" and s["kv"] == "q8":
        s["lk"], s["lv"] = (torch.empty(n, nkv * hd, **dev) for _ in range(2))


def _loaded(s, h, seq, row, table):
    """8-bit rows as the values that they stand for; others as the pages hold them"""
    if s["kv"] != "q8":
        return {"k": s["pool"]["k"][s.get("first", 0):], "v": s["pool"]["v"][s.get("first", 0):]}
    h.krh_paged_load(s["lk"].data_ptr(), s["lk"].shape[1], s["lv"].data_ptr(), s["lv"].shape[1], C.byref(s["pages"]),
                     table.data_ptr(), table.shape[1], s["seqs"], seq.numel(), seq.data_ptr(), row.data_ptr())
    return {"k": s["lk"], "v": s["lv"]}


def _run_own(s):
    h = _binding_of().hip
    if s["kind"] == "rules":
        v = s["vocab"]
        h.krh_logit_rules(s["out"].data_ptr(), v, s["logits"].data_ptr(), v, v, s["rows"], s["rule"].data_ptr(),
                          s["ids"].data_ptr(), s["ids"].shape[1], s["n_ids"].data_ptr(), s["bias_ids"].data_ptr(),
                          s["bias"].data_ptr(), s["bias"].shape[1], s["n_bias"].data_ptr(), s["bits"].data_ptr(),
                          s["bits"].shape[0])
        return s["out"]
    pages, table, ld = C.byref(s["pages"]), s["table"].data_ptr(), s["table"].shape[1]
    if s["kind"] == "attn":
        if s["mass"]:
            h.krh_copy_d2d_async(s["mass1"].data_ptr(), s["mass0"].data_ptr(), s["mass0"].nbytes)
        h.krh_paged_attention(s["o"].data_ptr(), pages, table, ld, s["len"].data_ptr(), s["seqs"], s["q"].data_ptr(),
                              s["heads"], s["rows"], s["window"], s["head_dim"] ** -0.5, s["softcap"],
                              _ptr(s["mass1"]), s["rows"], s["ws"].data_ptr())
        return {"o": s["o"], "mass": s["mass1"]} if s["mass"] else {"o": s["o"]}
    if s["kind"] == "qkv":
        h.krh_paged_qkv(s["qo"].data_ptr(), s["qo"].shape[1], pages, table, ld, s["seqs"], s["q"].data_ptr(),
                        s["q"].shape[1], s["k"].data_ptr(), s["k"].shape[1], s["v"].data_ptr(), s["v"].shape[1],
                        s["tokens"], s["heads"], s["seq"].data_ptr(), s["row"].data_ptr(), s["pos"].data_ptr(),
                        _ptr(s["qw"]), _ptr(s["kw"]), EPS, s["cos"].data_ptr(), s["sin"].data_ptr(),
                        s["cos"].shape[0])
        return {"q": s["qo"], **_loaded(s, h, s["seq"], s["row"], s["table"])}
    h.krh_paged_evict(pages, table, ld, s["len"].data_ptr(), s["weight"].data_ptr(), s["rows"], s["seqs"], s["rows"],
                      s["keep"], s["recent"], s["out_table"].data_ptr(), s["out_table"].shape[1],
                      s["len1"].data_ptr(), s["weight1"].data_ptr(), s["keep"], s["ws"].data_ptr())
    return {"len": s["len1"], "mass": s["weight1"], **_loaded(s, h, s["lseq"], s["lrow"], s["out_table"])}


def _binding_of():
    return sys.modules["krafla"]


# ---- the plain forms ----

def run(s):
    if own:
        return _run_own(s)
    return {"attn": _attn, "qkv": _qkv, "evict": _evict, "rules": _rules}[s["kind"]](s)


def _values(pool, n):
    """the pages' K or V in 32 bits"""
    x = pool[n].float()
    return x * pool[n + "d"].unsqueeze(-1) if n + "d" in pool else x


def _gathered(s, n):
    """[seq][kv head][row][dim] of the sequences' pages; what lies behind their rows is left out later"""
    t = s["table"].clamp(min=0).long()
    x = s["pool"][n][t].float()
    if n + "d" in s["pool"]:
        x = x * s["pool"][n + "d"][t].unsqueeze(-1)
    x = x.permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])[:, :, :s["rows"]].contiguous()


def _attn(s):
    n, nkv, hd = s["seqs"], s["kv_heads"], s["head_dim"]
    q = s["q"].view(n, nkv, -1, hd)
    z = torch.matmul(_gathered(s, "k"), q.transpose(2, 3).contiguous()) * hd ** -0.5   # [seq][kv head][row][head]
    if s["softcap"] > 0:
        z = s["softcap"] * torch.tanh(z / s["softcap"])
    row, ln = torch.arange(s["rows"], device="cuda").view(1, 1, -1, 1), s["len"].view(-1, 1, 1, 1)
    ok = row < ln
    if s["window"]:
        ok = ok & (row >= ln - s["window"])
    z = z.masked_fill(~ok, -math.inf)
    e = torch.exp(z - z.amax(2, keepdim=True))
    a = e / e.sum(2, keepdim=True)
    o = torch.matmul(a.transpose(2, 3).contiguous(), _gathered(s, "v")).view(n, -1, hd)
    return {"o": o, "mass": s["mass0"] + a.sum(3)} if s["mass"] else {"o": o}


def _norm_rotate(s, x, w):
    x = x.view(s["tokens"], -1, s["head_dim"])
    if w is not None:
        # the sum in 64 bits, so that an 8-bit value next to a border falls on one side of it
        x = x * (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float() * w
    c, sn = s["cos"][s["pos"].long()].unsqueeze(1), s["sin"][s["pos"].long()].unsqueeze(1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * sn, a * sn + b * c], -1).view(x.shape)


def _q8(x):
    """int8 rows of one scale each"""
    m = x.abs().amax(-1, keepdim=True)
    return torch.trunc(x * (127 / m) + torch.copysign(torch.full_like(x, 0.5), x)).clamp(-127, 127), m / 127


def _qkv(s):
    rows = [_norm_rotate(s, s["k"], s["kw"]), s["v"].view(s["tokens"], -1, s["head_dim"])]
    q = _norm_rotate(s, s["q"], s["qw"]).view(s["tokens"], -1)
    if s["kv"] == "q8":
        k, v = ((n * d).view(s["tokens"], -1) for n, d in map(_q8, rows))
        return {"q": q, "k": k, "v": v}
    row = s["row"].long()
    at = s["table"][s["seq"].long(), row // s["page"]].long(), row % s["page"]
    k, v = (torch.zeros_like(s["pool"][n]) for n in ("k", "v"))
    k[at[0], :, at[1]], v[at[0], :, at[1]] = rows[0].to(k.dtype), rows[1].to(v.dtype)
    return {"q": q, "k": k, "v": v}


def _evict(s):
    n, keep, R = s["seqs"], s["keep"], s["rows"]
    ln, row = s["len"].long().view(-1, 1, 1), torch.arange(R, device="cuda").view(1, 1, -1)
    key = torch.where(row >= ln - s["recent"], math.inf, s["weight"]).masked_fill(row >= ln, -math.inf)
    at = torch.sort(key, dim=2, descending=True, stable=True)[1][:, :, :keep]
    at = torch.sort(torch.where(at < ln, at, R), dim=2)[0]               # rows kept, in order; R past them
    new = ln.clamp(max=keep).view(-1)
    past, at = at >= R, at.clamp(max=R - 1)
    out = {"len": new.int(), "mass": torch.gather(s["weight"], 2, at).masked_fill(past, 0.0)}
    page = s["table"].long().gather(1, (at // s["page"]).view(n, -1)).view(at.shape).clamp(min=0)
    kvh = torch.arange(s["kv_heads"], device="cuda").view(1, -1, 1)
    i, j = s["lseq"].long(), s["lrow"].long()
    to = s["out_table"].long()[i, j // s["page"]] - s["first"], slice(None), j % s["page"]
    if s["kv"] == "q8":
        k, v = (s["pool"][m][page, kvh, at % s["page"]].float() * s["pool"][m + "d"][page, kvh, at % s["page"]].unsqueeze(-1)
                for m in ("k", "v"))
        return {**out, "k": k[i, :, j].reshape(i.numel(), -1), "v": v[i, :, j].reshape(i.numel(), -1)}
    k, v = (torch.zeros_like(s["pool"][m][s["first"]:]) for m in ("k", "v"))
    k[to] = s["pool"]["k"][page, kvh, at % s["page"]][i, :, j]
    v[to] = s["pool"]["v"][page, kvh, at % s["page"]][i, :, j]
    return {**out, "k": k, "v": v}


def _rules(s):
    r, v = s["rows"], s["vocab"]
    x = s["logits"]
    ids = s["ids"].long()
    ids = torch.where(torch.arange(ids.shape[1], device="cuda") < s["n_ids"].unsqueeze(1), ids, v)
    c = torch.zeros(r, v + 1, device="cuda").scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))[:, :v]
    rp = s["repeat"].unsqueeze(1)
    y = torch.where(x > 0, x / rp, x * rp) - s["frequency"].unsqueeze(1) * c - s["presence"].unsqueeze(1)
    x = torch.where(c > 0, y, x)
    at = torch.arange(s["bias_ids"].shape[1], device="cuda")
    ids = torch.where(at < s["n_bias"].unsqueeze(1), s["bias_ids"].long(), v)
    last = torch.full((r, v + 1), -1, device="cuda").scatter_reduce_(1, ids, at.expand(r, -1), "amax")[:, :v]
    x = torch.where(last >= 0, x + s["bias"].gather(1, last.clamp(min=0)), x)
    bits = (s["bits"].unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device="cuda") & 1).view(s["bits"].shape[0], -1)[:, :v]
    off = (bits[s["mask"].clamp(min=0).long()] == 0) & (s["mask"] >= 0).unsqueeze(1)
    return x.masked_fill(off, -math.inf)


# ---- what a pass cannot do without ----

def _row_bytes(case):
    """one row's K and V of all KV heads"""
    return case["kv_heads"] * (2 * case["head_dim"] * WIDTH[case["kv"]] + (8 if case["kv"] == "q8" else 0))


def work(case):
    kind = case["kind"]
    if kind == "rules":
        n = case["rows"] * case["vocab"]
        return dict(bytes=8 * n + 4 * case["rows"] * case["seen"] + (n // 16 if case["masks"] else 0), flops=2 * n)
    hd, nh, nkv = case["head_dim"], case["heads"], case["kv_heads"]
    if kind == "qkv":
        # 8 bits: the rows come back as the values that they stand for
        row = 8 * nh * hd + 8 * nkv * hd + _row_bytes(case) * (2 if case["kv"] == "q8" else 1) + 4 * hd
        row += 8 * nkv * hd if case["kv"] == "q8" else 0
        return dict(bytes=case["tokens"] * row, flops=case["tokens"] * (nh + nkv) * hd * (6 if case["norm"] else 3))
    lens = _lens(case, case["rows"])
    if kind == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        row = _row_bytes(case) * (3 if case["kv"] == "q8" else 2) + (8 * nkv * hd if case["kv"] == "q8" else 0)
        return dict(bytes=kept * row + 4 * nkv * (sum(lens) + case["seqs"] * case["keep"]), flops=nkv * sum(lens))
    n = sum(min(v, case["window"]) if case["window"] else v for v in lens)
    return dict(bytes=n * _row_bytes(case) + 8 * case["seqs"] * nh * hd + (8 * nkv * n if case["mass"] else 0),
                flops=4 * nh * hd * n)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _attn_exact, "qkv": _qkv_exact, "evict": _evict_exact, "rules": _rules_exact}[case["kind"]](s)


def _rows_exact(s, name, i, n):
    """[row][kv head][dim] of the first n rows of sequence i"""
    at = torch.arange(n, device="cuda")
    page, slot = s["table"][i].long()[at // s["page"]], at % s["page"]
    x = s["pool"][name][page, :, slot].double()
    if s["kv"] == "q8":
        x = x * s["pool"][name + "d"][page, :, slot].double().unsqueeze(-1)
    return x


def _attn_exact(s):
    nkv, hd = s["kv_heads"], s["head_dim"]
    o = torch.zeros(s["seqs"], s["heads"], hd, dtype=torch.float64, device="cuda")
    mass = s["mass0"].double().clone() if s["mass"] else None
    for i, n in enumerate(s["len"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        k, v = _rows_exact(s, "k", i, n)[first:], _rows_exact(s, "v", i, n)[first:]
        for g in range(nkv):
            h = slice(g * s["heads"] // nkv, (g + 1) * s["heads"] // nkv)
            z = s["q"][i, h].double() @ k[:, g].t().contiguous() / math.sqrt(hd)
            if s["softcap"] > 0:
                z = s["softcap"] * torch.tanh(z / s["softcap"])
            a = torch.softmax(z, 1)
            o[i, h] = a @ v[:, g].contiguous()
            if mass is not None:
                mass[i, g, first:n] += a.sum(0)
    return {"o": o, "mass": mass} if s["mass"] else {"o": o}


def _qkv_exact(s):
    T, hd = s["tokens"], s["head_dim"]

    def turned(x, w):
        x = x.double().view(T, -1, hd)
        if w is not None:
            x = x / torch.sqrt((x * x).sum(2, keepdim=True) / hd + EPS) * w.double()
        z = torch.view_as_complex(x.view(T, x.shape[1], hd // 2, 2).contiguous())
        p = s["pos"].long()
        return torch.view_as_real(z * torch.complex(s["cos"][p].double(), s["sin"][p].double()).unsqueeze(1)).reshape(T, -1)

    q, k, v = turned(s["q"], s["qw"]), turned(s["k"], s["kw"]), s["v"].double()
    if s["kv"] == "q8":
        # which of two 8-bit values holds is decided by the rule's 32-bit
        # products, so what they stand for has no other form in 64 bits
        return {"q": q, "k": None, "v": None}
    out = {"q": q}
    for name, x in (("k", k), ("v", v)):
        y = torch.zeros(s["pool"][name].shape, dtype=torch.float64, device="cuda")
        page = s["table"][s["seq"].long(), s["row"].long() // s["page"]].long()
        y[page, :, s["row"].long() % s["page"]] = x.view(T, -1, hd)
        out[name] = y
    return out


def _evict_exact(s):
    # which rows stay is decided by comparisons of the weights as they are, so
    # the values that follow have no other form in 64 bits
    keep, R, weight = s["keep"], s["recent"], s["weight"].cpu()
    mass = torch.zeros(s["seqs"], s["kv_heads"], keep, dtype=torch.float64)
    for i, n in enumerate(s["len"].tolist()):
        for g in range(s["kv_heads"]):
            w = weight[i, g, :n].tolist()
            if n > keep:
                old = sorted(range(n - R), key=lambda r: (-w[r], r))[:keep - R]
                w = [w[r] for r in sorted(old)] + w[n - R:]
            mass[i, g, :len(w)] = torch.tensor(w, dtype=torch.float64)
    return {"len": None, "mass": mass, "k": None, "v": None}


def _rules_exact(s):
    x = s["logits"].double().cpu()
    ids, n_ids, b_ids, n_bias, bias = (s[n].cpu() for n in ("ids", "n_ids", "bias_ids", "n_bias", "bias"))
    repeat, presence, frequency, mask, words = (s[n].cpu() for n in ("repeat", "presence", "frequency", "mask", "bits"))
    for i in range(s["rows"]):
        c = torch.bincount(ids[i, :n_ids[i]].long(), minlength=s["vocab"]).double()
        seen = c.nonzero().view(-1)
        rp = repeat[i].double()
        y = x[i, seen]
        y = torch.maximum(y, torch.zeros_like(y)) / rp + torch.minimum(y, torch.zeros_like(y)) * rp
        x[i, seen] = y - frequency[i].double() * c[seen] - presence[i].double()
        for t, b in {int(t): float(b) for t, b in zip(b_ids[i, :n_bias[i]], bias[i])}.items():
            x[i, t] += b
        if mask[i] >= 0:
            at = torch.arange(s["vocab"])
            x[i, (words[mask[i]].long()[at // 32] >> (at % 32)) & 1 == 0] = -math.inf
    return x


if __name__ == "__main__":
    for number in range(6):
        print(draw(random.Random(number)))
