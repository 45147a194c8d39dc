"""Several continuations of one prompt, as calls that can be timed and compared.

The operators a program needs that keeps the prompt's KV cache once and decodes many answers from it:

  logprobs   log probabilities of given tokens with the row's logsumexp, entropy and most probable alternatives
  copy       pages of a paged KV cache copied for all layers at once: a fork's last page, a compaction
  append     q / k norm, rotary positions and the write of a batch's new rows into its pages
  attention  a batch of sequences that share a long prefix, over pages, with the output gate

Shapes are those of the full-attention layers of the model this library serves (16 query heads on 2
KV heads of 256, ten such layers, a vocabulary of 248320 and a draft vocabulary of 32768), or generic.
Where `own` is false everything is elementary torch arithmetic. Where it is true the calls run on the stream of the library's own
context, which is not ordered with torch's: `prepare` waits until torch has made the inputs, and who reads a pass's outputs, times it or
changes its inputs waits for the whole device first (torch.cuda.synchronize()).
"""
import ctypes as C
import importlib
import math

import numpy as np
import torch

own = False

V, DRAFT_V, LAYERS, HQ, HKV, HD, ROPE = 248320, 32768, 10, 16, 2, 256, 64
EPS, THETA = 1e-6, 1e7


# ---- cases ---------------------------------------------------------------------------------
def listed():
    return [
        # one sampled token of a chat reply, with the twenty alternatives an API may be asked for
        dict(name="logprobs-1", op="logprobs", rows=1, V=V, given=1, k=20, dtype="bf16", masked=0.0),
        # four draft rows over the reduced vocabulary, under a grammar that leaves one token in twenty
        dict(name="logprobs-4-draft-grammar", op="logprobs", rows=4, V=DRAFT_V, given=3, k=5, dtype="f32", masked=0.95),
        # scoring a page of text
        dict(name="logprobs-700", op="logprobs", rows=700, V=V, given=1, k=8, dtype="bf16", masked=0.0),
        # three more answers from one prompt: its last, partly filled page for all layers
        dict(name="copy-fork-3", op="copy", pages=64, page_rows=64, src=1, copies=3, rows=29, layers=LAYERS, Hkv=HKV, hd=HD),
        # a compaction of a pool that many answers have come and gone in
        dict(name="copy-compact-240", op="copy", pages=640, page_rows=64, src=240, copies=1, rows=64, layers=LAYERS, Hkv=HKV, hd=HD),
        # eight answers, one new token each
        dict(name="append-8x1", op="append", B=8, T=1, rows=180, page_rows=64, Hq=HQ, Hkv=HKV, hd=HD, rope=ROPE),
        # 64 answers with three drafts each to verify
        dict(name="append-64x4", op="append", B=64, T=4, rows=250, page_rows=64, Hq=HQ, Hkv=HKV, hd=HD, rope=ROPE),
        # four answers to a short question, just begun
        dict(name="attention-4x1-at-60", op="attention", B=4, T=1, shared=0, rows=60, page_rows=64, Hq=HQ, Hkv=HKV, hd=HD),
        # eight answers about a long document
        dict(name="attention-8x1-at-6621", op="attention", B=8, T=1, shared=6592, rows=200, page_rows=64, Hq=HQ, Hkv=HKV, hd=HD),
        # four answers with one draft each, small pages, eight KV heads of 128
        dict(name="attention-4x2-at-2000-heads8", op="attention", B=4, T=2, shared=1984, rows=333, page_rows=16, Hq=32, Hkv=8, hd=128),
        # sixteen answers at the end of a long context, depth-3 verification
        dict(name="attention-16x4-at-16300", op="attention", B=16, T=4, shared=16256, rows=77, page_rows=64, Hq=HQ, Hkv=HKV, hd=HD),
        # 64 of them behind twice that context
        dict(name="attention-64x4-at-32768", op="attention", B=64, T=4, shared=32768, rows=512, page_rows=64, Hq=HQ, Hkv=HKV, hd=HD),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 2, 256), (16, 2, 256), (16, 2, 256), (32, 8, 128), (16, 16, 128), (24, 2, 128), (8, 1, 64), (12, 4, 64), (6, 2, 256)]


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "copy", "append", "attention", "attention", "attention"])
    if op == "logprobs":
        v = rng.choice([V, DRAFT_V, _log(rng, 50, 250000)])
        rows = max(1, min(_log(rng, 1, 700), 700 * V // v))
        dtype = rng.choice(["bf16", "f32"])
        return dict(op=op, rows=rows if dtype == "bf16" else max(1, rows // 2), V=v, given=rng.choice([1, 1, 2, 7]), k=min(v, rng.randint(0, 32)),
                    dtype=dtype, masked=rng.choice([0.0, 0.0, 0.5, 0.999]))
    hq, hkv, hd = rng.choice(HEADS)
    R = rng.choice([16, 32, 64, 128, 256])
    if op == "copy":
        src, copies, layers = _log(rng, 1, 200), rng.choice([1, 1, 2, 7]), rng.randint(1, LAYERS)
        while src * copies * R > 240 * 64:
            src = src // 2 + 1
            copies = 1
        return dict(op=op, pages=src * (copies + 1) + rng.randint(0, 50), page_rows=R, src=src, copies=copies, rows=rng.randint(1, R),
                    layers=layers, Hkv=hkv, hd=hd)
    if op == "append":
        T = rng.randint(1, 8)
        return dict(op=op, B=_log(rng, 1, 64), T=T, rows=T + _log(rng, 1, 250), page_rows=R, Hq=hq, Hkv=hkv, hd=hd, rope=rng.choice([hd // 4, hd // 2, hd]))
    while True:
        T = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
        c = dict(op=op, B=_log(rng, 1, 64), T=T, shared=rng.choice([0, 1, 1, 1]) * (_log(rng, 16, 32768) // R * R), rows=T + _log(rng, 1, 1500),
                 page_rows=R, Hq=hq, Hkv=hkv, hd=hd)
        w, most = work(c), work(listed()[-1])
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return c


def _lens(c):
    """Rows that each sequence holds: the shared ones and between half and all of `rows` own ones (at least T)."""
    own_rows = [max(c["T"], c["rows"] - (b * c["rows"] // 2) // c["B"]) for b in range(c["B"])]
    return [c.get("shared", 0) + n for n in own_rows]


def work(c):
    if c["op"] == "logprobs":
        n = c["rows"] * c["V"]
        return {"bytes": n * (2 if c["dtype"] == "bf16" else 4) + c["rows"] * (8 + 8 * c["given"] + 8 * c["k"]), "flops": 6.0 * n}
    if c["op"] == "copy":
        page = 2 * c["layers"] * c["Hkv"] * c["rows"] * c["hd"] * 2
        return {"bytes": page * (c["src"] + c["src"] * c["copies"]), "flops": 0}
    B, T, hq, hkv, hd = (c[n] for n in ("B", "T", "Hq", "Hkv", "hd"))
    if c["op"] == "append":
        return {"bytes": 2 * B * T * (hq + 2 * hkv) * hd * 2 + B * T * (c["rope"] * 4 + 8), "flops": B * T * (hq + hkv) * (4.0 * hd + 3 * c["rope"])}
    keys = c["shared"] + sum(n - c["shared"] for n in _lens(c))
    seen = sum(n - T + t + 1 for n in _lens(c) for t in range(T))
    return {"bytes": 2 * hkv * keys * hd * 2 + 3 * B * T * hq * hd * 2, "flops": 4.0 * seen * hq * hd}


# ---- inputs ----------------------------------------------------------------------------------
class _Buf:
    """A torch tensor where the binding expects one of its device buffers."""

    def __init__(self, t):
        self.t, self.ptr = t, C.c_void_p(t.data_ptr())


class _State:
    def __init__(self, case):
        self.case = case


def _normal(g, shape, std=1.0, mean=0.0):
    return _Buf((torch.randn(shape, generator=g, device="cuda") * std + mean).to(torch.bfloat16))


def _empty(shape, dtype=torch.bfloat16):
    return _Buf(torch.empty(shape, device="cuda", dtype=dtype))


def prepare(case, seed):
    s, g = _State(case), torch.Generator(device="cuda")
    g.manual_seed(seed)
    {"logprobs": _prep_logprobs, "copy": _prep_copy, "append": _prep_append, "attention": _prep_attention}[case["op"]](s, case, g)
    if own:
        torch.cuda.synchronize()  # (another stream than torch's reads them)
    return s


def _prep_logprobs(s, c, g):
    rows, v = c["rows"], c["V"]
    x = torch.randn((rows, v), generator=g, device="cuda") * 2.5
    # one row in two is sure of a token, as most positions of a text are
    top = torch.randint(0, v, (rows,), generator=g, device="cuda")
    x[torch.arange(0, rows, 2, device="cuda"), top[::2]] += 16.0
    if c["masked"]:
        off = torch.rand((rows, v), generator=g, device="cuda") < c["masked"]
        off[torch.arange(rows, device="cuda"), top] = False
        x.masked_fill_(off, -math.inf)
    s.x = _Buf(x.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32))
    given = torch.randint(0, v, (rows, c["given"]), generator=g, device="cuda", dtype=torch.int32)
    given[:, 0] = top.to(torch.int32)
    s.given = _Buf(given)
    s.lp, s.ent, s.lse = _empty((rows, c["given"]), torch.float32), _empty((rows,), torch.float32), _empty((rows,), torch.float32)
    s.ids, s.tlp = _empty((rows, max(c["k"], 1)), torch.int32), _empty((rows, max(c["k"], 1)), torch.float32)


def _pools(s, c, g, pages, layers):
    s.k = _normal(g, (layers, pages, c["Hkv"], c["page_rows"], c["hd"]))
    s.v = _normal(g, (layers, pages, c["Hkv"], c["page_rows"], c["hd"]))
    s.pages = pages


def _prep_copy(s, c, g):
    _pools(s, c, g, c["pages"], c["layers"])
    order = torch.randperm(c["pages"], generator=g, device="cuda").to(torch.int32).cpu()
    n = c["src"]
    src, dst = order[:n].repeat_interleave(c["copies"]), order[n:n + n * c["copies"]]
    s.src, s.dst = src.numpy().astype(np.uint32), dst.numpy().astype(np.uint32)       # a pool's bookkeeping is on the host
    s.src_ids, s.dst_ids = src.cuda().long(), dst.cuda().long()


def _table(s, c, g, shared):
    """Page tables of B sequences whose first `shared` rows are the same pages, in no order."""
    B, R = c["B"], c["page_rows"]
    lens, ns = _lens(c), shared // R
    most = (max(lens) + R - 1) // R
    _pools(s, c, g, ns + B * (most - ns), 1)
    ids = torch.randperm(s.pages, generator=g, device="cuda").to(torch.int32)
    s.table = _Buf(torch.cat([ids[:ns].expand(B, ns), ids[ns:].reshape(B, most - ns)], 1).contiguous())
    s.lens = _Buf(torch.tensor(lens, dtype=torch.int32, device="cuda"))
    s.most, s.max_rows = most, max(lens)


def _prep_append(s, c, g):
    _table(s, c, g, 0)
    B, T, hq, hkv, hd = (c[n] for n in ("B", "T", "Hq", "Hkv", "hd"))
    s.qg, s.kx, s.vx = _normal(g, (B, T, hq, 2 * hd)), _normal(g, (B, T, hkv, hd)), _normal(g, (B, T, hkv, hd))
    s.qw, s.kw = _normal(g, (hd,), 0.1, 1.0), _normal(g, (hd,), 0.1, 1.0)
    half = c["rope"] // 2
    s.npos = s.max_rows
    ang = torch.arange(s.npos, device="cuda", dtype=torch.float64)[:, None] * THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    s.cos, s.sin = _Buf(ang.cos().float()), _Buf(ang.sin().float())
    s.q = _empty((B, T, hq, hd))


def _prep_attention(s, c, g):
    _table(s, c, g, c["shared"])
    B, T, hq, hd = (c[n] for n in ("B", "T", "Hq", "hd"))
    s.q, s.qg, s.out = _normal(g, (B, T, hq, hd), 2.0), _normal(g, (B, T, hq, 2 * hd)), _empty((B, T, hq, hd))


# ---- one pass --------------------------------------------------------------------------------
def run(s):
    return {"logprobs": _run_logprobs, "copy": _run_copy, "append": _run_append, "attention": _run_attention}[s.case["op"]](s)


_lib = None


def _own():
    """(the binding package, a context), made on first use and kept as a program keeps them."""
    global _lib
    if _lib is None:
        orn = importlib.import_module("ornith-rs_amd")
        _lib = orn, orn.Ctx(0)
    return _lib


def _kv(s):
    """The pages' and the batch's descriptors, which a program keeps with its pool."""
    if not hasattr(s, "kv"):
        orn, c = _own()[0], s.case
        layers = [(_Buf(s.k.t[i]), _Buf(s.v.t[i])) for i in range(s.k.t.shape[0])]
        s.kv = orn.KvPages([k for k, _ in layers], [v for _, v in layers], s.pages, c["page_rows"], c["Hkv"], c["hd"])
        if hasattr(s, "table"):
            s.batch = orn.KvBatch(c["B"], s.table, s.most, s.lens, c.get("shared", 0), s.max_rows)
    return s.kv


def _run_logprobs(s):
    c = s.case
    if own:
        orn, ctx = _own()
        ctx.token_logprobs(s.x, orn.BF16 if c["dtype"] == "bf16" else orn.F32, c["rows"], c["V"], s.given, c["given"], c["k"], s.lp, s.ent, s.lse,
                           s.ids, s.tlp)
        out = [s.lp.t, s.ent.t, s.lse.t]
        return out + [s.ids.t, s.tlp.t] if c["k"] else out
    x = s.x.t.float()
    m = x.max(1, keepdim=True).values
    d = x - m
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    lp = d.gather(1, s.given.t.long()) - log_total
    ent = log_total - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total
    out = [lp, ent[:, 0], (m + log_total)[:, 0]]
    if c["k"]:
        ids = s.x.t.sort(dim=1, descending=True, stable=True).indices[:, :c["k"]]
        out += [ids.to(torch.int32), d.gather(1, ids) - log_total]
    return out


def _run_copy(s):
    c = s.case
    if own:
        _own()[1].kv_pages_copy(_kv(s), s.src, s.dst, c["rows"])
    else:
        src, dst = s.src_ids, s.dst_ids
        s.k.t[:, dst, :, :c["rows"]] = s.k.t[:, src, :, :c["rows"]]
        s.v.t[:, dst, :, :c["rows"]] = s.v.t[:, src, :, :c["rows"]]
    return [s.k.t, s.v.t]


def _rotate(x, cos, sin, half):
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _run_append(s):
    c = s.case
    if own:
        _own()[1].attn_prep_paged(_kv(s), 0, s.batch, s.qg, s.kx, s.vx, s.qw, s.kw, c["T"], c["Hq"], c["rope"], EPS, s.cos, s.sin, s.npos, s.q)
        return [s.q.t, s.k.t, s.v.t]
    T, R, half = c["T"], c["page_rows"], c["rope"] // 2
    pos = s.lens.t.long()[:, None] - T + torch.arange(T, device="cuda")
    page, row = s.table.t.long().gather(1, pos // R), pos % R
    cos, sin = s.cos.t[pos][:, :, None], s.sin.t[pos][:, :, None]

    def normed(x, w):
        x = x.float()
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()

    s.q.t.copy_(_rotate(normed(s.qg.t[..., :c["hd"]], s.qw.t), cos, sin, half))
    s.k.t[0][page, :, row] = _rotate(normed(s.kx.t, s.kw.t), cos, sin, half).to(torch.bfloat16)
    s.v.t[0][page, :, row] = s.vx.t
    return [s.q.t, s.k.t, s.v.t]


def _run_attention(s):
    c = s.case
    if own:
        _own()[1].sdpa_paged_gated(_kv(s), 0, s.batch, s.q, s.qg, c["T"], c["Hq"], c["hd"] ** -0.5, s.out)
        return s.out.t
    B, T, hq, hkv, hd, R = (c[n] for n in ("B", "T", "Hq", "Hkv", "hd", "page_rows"))
    G, S, ns = hq // hkv, c["shared"], c["shared"] // R
    q = s.q.t.float().reshape(B, T, hkv, G, hd).permute(2, 0, 1, 3, 4) * hd ** -0.5          # [hkv, B, T, G, hd]
    table = s.table.t.long()

    def rows(pool, ids):                                                                     # [.., hkv, rows, hd]
        x = pool[0][ids].float().movedim(-3, -4)
        return x.reshape(x.shape[:-3] + (x.shape[-3] * R, hd)).contiguous()

    own_k, own_v = rows(s.k.t, table[:, ns:]), rows(s.v.t, table[:, ns:])                    # [B, hkv, n, hd]
    n = own_k.shape[2]
    sc = torch.matmul(q.permute(1, 0, 2, 3, 4).reshape(B, hkv, T * G, hd), own_k.transpose(2, 3).contiguous()).reshape(B, hkv, T, G, n)
    pos = s.lens.t.long()[:, None] - T + torch.arange(T, device="cuda")
    hidden = torch.arange(S, S + n, device="cuda") > pos[:, :, None]                         # [B, T, n]
    sc.masked_fill_(hidden[:, None, :, None], -math.inf)
    m = sc.max(-1, keepdim=True).values
    if S:
        sh_k, sh_v = rows(s.k.t, table[0, :ns]), rows(s.v.t, table[0, :ns])                  # [hkv, S, hd]
        sh = torch.matmul(q.reshape(hkv, B * T * G, hd), sh_k.transpose(1, 2).contiguous())  # [hkv, B T G, S]
        sh_m = sh.max(-1, keepdim=True).values.reshape(hkv, B, T, G, 1).movedim(0, 1)
        m = torch.maximum(m, sh_m)
        sh = (sh - m.movedim(1, 0).reshape(hkv, B * T * G, 1)).exp()
    p = (sc - m).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, hkv, T * G, n), own_v).reshape(B, hkv, T, G, hd)
    if S:
        total = total + sh.sum(-1, keepdim=True).reshape(hkv, B, T, G, 1).movedim(0, 1)
        o = o + torch.matmul(sh, sh_v).reshape(hkv, B, T, G, hd).movedim(0, 1)
    o = (o / total).permute(0, 2, 1, 3, 4).reshape(B, T, hq, hd)
    return (o / (1 + (-s.qg.t[..., hd:].float()).exp())).to(torch.bfloat16)


# ---- in 64 bits ------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "copy": _exact_copy, "append": _exact_append, "attention": _exact_attention}[case["op"]](s, case)


def _exact_logprobs(s, c):
    got = []
    for r in range(c["rows"]):
        x = s.x.t[r].double()
        lse = torch.logsumexp(x, 0)
        p = torch.exp(x - lse)
        some = p > 0
        row = [x[s.given.t[r].long()] - lse, -(p[some] * (x[some] - lse)).sum(), lse]
        if c["k"]:
            # one key a token, larger for a larger value and, among equals, for a lower index
            bits = s.x.t[r].float().view(torch.int32).long() + 0
            bits = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
            key = bits * (1 << 20) + (c["V"] - 1 - torch.arange(c["V"], device="cuda"))
            ids = torch.topk(key, c["k"]).indices
            row += [ids.to(torch.int32), x[ids] - lse]
        got.append(row)
    return [torch.stack(col) for col in zip(*got)]


def _exact_copy(s, c):
    for pool in (s.k.t, s.v.t):
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            pool[:, b, :, :c["rows"]] = pool[:, a, :, :c["rows"]]
    return [s.k.t.double(), s.v.t.double()]


def _exact_append(s, c):
    T, R, hd, half = c["T"], c["page_rows"], c["hd"], c["rope"] // 2
    q = torch.empty((c["B"], T, c["Hq"], hd), device="cuda", dtype=torch.float64)
    k, v = s.k.t.double(), s.v.t.double()
    table, lens = s.table.t.tolist(), s.lens.t.tolist()

    def head(x, w, pos):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = torch.complex(y[:, :half], y[:, half:2 * half]) * torch.complex(s.cos.t[pos].double(), s.sin.t[pos].double())
        return torch.cat([z.real, z.imag, y[:, 2 * half:]], 1)

    for b in range(c["B"]):
        for t in range(T):
            pos = lens[b] - T + t
            q[b, t] = head(s.qg.t[b, t, :, :hd], s.qw.t, pos)
            k[0, table[b][pos // R], :, pos % R] = head(s.kx.t[b, t], s.kw.t, pos)
            v[0, table[b][pos // R], :, pos % R] = s.vx.t[b, t].double()
    return [q, k, v]


def _exact_attention(s, c):
    B, T, hq, hkv, hd = (c[n] for n in ("B", "T", "Hq", "Hkv", "hd"))
    out = torch.empty((B, T, hq, hd), device="cuda", dtype=torch.float64)
    table, lens = s.table.t.long(), s.lens.t.tolist()
    for b in range(B):
        k = s.k.t[0][table[b]].double().transpose(0, 1).reshape(hkv, -1, hd)
        v = s.v.t[0][table[b]].double().transpose(0, 1).reshape(hkv, -1, hd)
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            keys, vals = k[h, :lens[b]].contiguous(), v[h, :lens[b]].contiguous()
            sc = torch.mm(s.q.t[b, :, heads].double().reshape(-1, hd), keys.t().contiguous()).reshape(T, -1, lens[b]) / math.sqrt(hd)
            for t in range(T):
                sc[t, :, lens[b] - T + t + 1:] = -math.inf
            att = torch.mm(torch.softmax(sc, -1).reshape(-1, lens[b]), vals).reshape(T, -1, hd)
            out[b, :, heads] = torch.sigmoid(s.qg.t[b, :, heads, hd:].double()) * att
    return out
