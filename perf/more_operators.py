"""What is measured of one prompt with many continuations and of a cache of bounded size, over
the binary16 KV cache: the cases, the operators' plain forms and their values in 64 bits.

Four operators, each through the entry points of hvdrv.py that a program calls:

  shared  attention of a batch of sequences that share a prefix, each with a tail of its own and
          one or more query rows (attn_shared)
  tails   the rows of such a batch written: head norms, rotation, K and V into the tails
          (qk_shared)
  mass    causal attention that also adds up the weight every cached position gets
          (attn_decode_mass for one token, attn_rows_mass for a run)
  evict   a cache thinned to the positions with the most weight and the latest ones (kv_evict)
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False          # set by the tools: True makes the calls of the framework's kernels

HD = 128
EPS = 1e-5
_PKG = str(Path(__file__).resolve().parent.parent / "hive-limited_b200")


def listed():
    return [
        # two answers to a short question under way: 16 q heads over 8 kv heads
        dict(name="shared-2-at-45", op="shared", nkv=8, group=2, nseq=2, prefix=45, tail_lo=1,
             tail_hi=9, rows_lo=1, rows_hi=1),
        # sixteen answers to one 4096-token document, one token each, 32 q heads over 8
        dict(name="shared-16-at-4096", op="shared", nkv=8, group=4, nseq=16, prefix=4096,
             tail_lo=1, tail_hi=256, rows_lo=1, rows_hi=1),
        # continuations of 3 to 17 tokens scored after a 2000-token prompt: ragged runs
        dict(name="shared-runs-24-at-2000", op="shared", nkv=8, group=4, nseq=24, prefix=2000,
             tail_lo=3, tail_hi=17, rows_lo=3, rows_hi=17),
        # the largest batch over the longest prefix
        dict(name="shared-64-at-32768", op="shared", nkv=8, group=4, nseq=64, prefix=32768,
             tail_lo=1, tail_hi=512, rows_lo=1, rows_hi=1),
        # a decode step's rows of sixteen sequences
        dict(name="tails-16", op="tails", nkv=8, group=4, nseq=16, prefix=4096, tail_lo=1,
             tail_hi=256, rows_lo=1, rows_hi=1),
        # the first run of 24 continuations, 64 q heads over 8
        dict(name="tails-runs-24", op="tails", nkv=8, group=8, nseq=24, prefix=2000, tail_lo=3,
             tail_hi=17, rows_lo=3, rows_hi=17),
        # one decode step inside the 4096 + 256 token workload
        dict(name="mass-decode-4225", op="mass", nkv=8, group=4, pos0=4224, ntok=1),
        # a decode step over a long cache, 64 q heads over 8
        dict(name="mass-decode-39999", op="mass", nkv=8, group=8, pos0=39998, ntok=1),
        # the second run of a 300-token prompt, 16 over 8
        dict(name="mass-44-at-256", op="mass", nkv=8, group=2, pos0=256, ntok=44),
        # a run deep in a 16k prompt, 64 over 8
        dict(name="mass-256-at-16128", op="mass", nkv=8, group=8, pos0=16128, ntok=256),
        # one layer of a small model, 300 positions to 256
        dict(name="evict-300-to-256", op="evict", nkv=2, nset=1, n=300, keep=256, recent=32),
        # the 36 layers of a model whose cache of 4352 positions is full, thinned to 4096
        dict(name="evict-36x4352-to-4096", op="evict", nkv=8, nset=36, n=4352, keep=4096,
             recent=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "shared", "tails", "mass", "mass", "mass", "evict",
                     "evict"])
    nkv = rng.choice([1, 2, 4, 8])
    if op == "evict":
        n = _log(rng, 2, 60000)
        keep = rng.randint(max(1, n // 8), n)
        return dict(op=op, nkv=nkv, nset=_log(rng, 1, max(1, min(36, 150000 // n))), n=n,
                    keep=keep, recent=rng.randint(0, keep))
    group = rng.randint(1, 8)
    if op == "mass":
        if rng.random() < 0.5:
            return dict(op=op, nkv=nkv, group=group, pos0=_log(rng, 1, 65536) - 1, ntok=1)
        return dict(op=op, nkv=nkv, group=group, pos0=_log(rng, 1, 16000) - 1,
                    ntok=_log(rng, 2, 256))
    prefix = 0 if rng.random() < 0.05 else _log(rng, 1, 32768)
    if rng.random() < 0.65:
        nseq, group = _log(rng, 1, 64), min(group, 4) if prefix > 16000 else group
        return dict(op=op, nkv=nkv, group=group, nseq=nseq, prefix=prefix,
                    tail_lo=1, tail_hi=_log(rng, 1, 512), rows_lo=1, rows_hi=1)
    most = _log(rng, 2, 40)
    least = rng.randint(1, most)
    return dict(op=op, nkv=nkv, group=group, nseq=rng.randint(1, min(64, 256 // most)),
                prefix=min(prefix, 8000), tail_lo=least, tail_hi=most + _log(rng, 1, 100),
                rows_lo=least, rows_hi=most)


def _lengths(case):
    """Rows and tail length (those rows among them) of every sequence."""
    spread = lambda i, a, b, m: a + (i * m + 17) % 97 * (b - a) // 96  # noqa: E731
    rows = [spread(i, case["rows_lo"], case["rows_hi"], 41) for i in range(case["nseq"])]
    tails = [max(r, spread(i, case["tail_lo"], case["tail_hi"], 59)) for i, r in enumerate(rows)]
    return rows, tails


def work(case):
    """Each input read once and each output written once: K and V 2 bytes a value, the rest 4.
    Attention: 4 * 128 operations for each (row, head, position) that is seen, and 128 * 2 more
    where the weights are formed again from the rows' sums (a run with mass)."""
    nkv, op = case["nkv"], case["op"]
    if op == "evict":
        n, keep, sets = case["n"], case["keep"], case["nset"] * nkv
        return {"bytes": sets * (4 * n + keep * (2 * 2 * 2 * HD + 4 + 4)), "flops": sets * 8 * n}
    nq = nkv * case["group"]
    if op == "mass":
        n, ntok = case["pos0"] + case["ntok"], case["ntok"]
        seen = ntok * n - ntok * (ntok - 1) // 2
        return {"bytes": nkv * n * (2 * 2 * HD + 8) + 2 * ntok * nq * HD * 4,
                "flops": nq * seen * HD * (4 if ntok == 1 else 6)}
    rows, tails = _lengths(case)
    if op == "tails":
        return {"bytes": sum(rows) * HD * (4 * (nq + 2 * nkv) + 4 * nq + 2 * 2 * nkv),
                "flops": sum(rows) * (nq + nkv) * HD * 8}
    seen = sum(r * (case["prefix"] + t) - r * (r - 1) // 2 for r, t in zip(rows, tails))
    return {"bytes": 2 * 2 * HD * nkv * (case["prefix"] + sum(tails)) + 2 * sum(rows) * nq * HD * 4,
            "flops": 4 * HD * nq * seen}


# ---- inputs --------------------------------------------------------------------------

def _cache(gen, *shape):
    """K and V rows [.., positions, 128] in binary16 as a model writes them: keys of unit scale
    after their norm with some dimensions larger, values a little smaller."""
    k = torch.randn(*shape, HD, generator=gen, device="cuda")
    k *= torch.exp(0.3 * torch.randn(HD, generator=gen, device="cuda"))
    v = 0.7 * torch.randn(*shape, HD, generator=gen, device="cuda") + 0.1
    return k.half(), v.half()


def _queries(gen, rows, nkv, group, k):
    """Queries that look for some of the positions k [nkv, n, 128], so that weights are not
    flat."""
    q = torch.randn(rows, nkv, group, HD, generator=gen, device="cuda")
    if k.shape[1]:
        at = torch.randint(0, k.shape[1], (rows, nkv, 4), generator=gen, device="cuda")
        look = k.float()[torch.arange(nkv, device="cuda")[None, :, None], at].mean(2)
        q += 0.8 * look[:, :, None]
    return q.reshape(rows, nkv * group, HD).contiguous()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    nkv, op = case["nkv"], case["op"]
    if op == "evict":
        n, keep, nset = case["n"], case["keep"], case["nset"]
        s["k"] = torch.empty(nset, nkv, n, HD, dtype=torch.float16, device="cuda")
        s["v"] = torch.empty_like(s["k"])
        for i in range(nset):
            s["k"][i], s["v"][i] = _cache(gen, nkv, n)
        # weights as they add up: a few positions have most, many have next to none
        m = torch.exp(2.0 * torch.randn(nset, nkv, n, generator=gen, device="cuda"))
        s["mass"] = torch.where(torch.rand(nset, nkv, n, generator=gen, device="cuda") < 0.2,
                                torch.zeros_like(m), m)
        s["len"] = _i32([n])
        s["out"] = [torch.zeros(nset, nkv, keep, HD, dtype=torch.float16, device="cuda"),
                    torch.zeros(nset, nkv, keep, HD, dtype=torch.float16, device="cuda"),
                    torch.zeros(nset, nkv, keep, device="cuda"),
                    torch.zeros(nset, nkv, keep, dtype=torch.int32, device="cuda"), _i32([0])]
        return s
    group = case["group"]
    nq = nkv * group
    s["scale"] = torch.tensor([1.0 / math.sqrt(HD)], device="cuda")
    if op == "mass":
        n, ntok = case["pos0"] + case["ntok"], case["ntok"]
        cap = s["cap"] = n + n % 7                       # a few rows of an older text behind it
        s["k"], s["v"] = _cache(gen, nkv, cap)
        s["q"] = _queries(gen, ntok, nkv, group, s["k"][:, :n])
        s["mass"] = torch.zeros(nkv, cap, device="cuda")
        s["mass"][:, :case["pos0"]] = torch.exp(torch.randn(nkv, case["pos0"], generator=gen,
                                                            device="cuda"))
        s["pos"] = _i32([n - 1])
        s["out"] = [torch.zeros(ntok, nq, HD, device="cuda"), torch.zeros(nkv, cap, device="cuda")]
        return s
    rows, tails = _lengths(case)
    s["nrow"], s["tcap"] = sum(rows), max(tails) + max(tails) % 3
    s["row_list"], s["tail_list"] = rows, tails
    s["row0"] = _i32(np.concatenate([[0], np.cumsum(rows)]).tolist())
    s["tlen"] = _i32(tails)
    s["tk"], s["tv"] = _cache(gen, case["nseq"], nkv, s["tcap"])
    seq = torch.repeat_interleave(torch.arange(case["nseq"]), torch.tensor(rows))
    slot = torch.cat([torch.arange(t - r, t) for r, t in zip(rows, tails)])
    s["seq"], s["slot"] = seq.cuda(), slot.cuda()
    if op == "tails":
        cap = case["prefix"] + s["tcap"]
        s["cap"], s["base"] = cap, _i32([case["prefix"]])
        ang = (np.arange(cap, dtype=np.float64)[:, None]
               / 1e6 ** (np.arange(HD // 2, dtype=np.float64) * 2.0 / HD)[None])
        s["cos"] = torch.from_numpy(np.cos(ang).astype(np.float32)).cuda()
        s["sin"] = torch.from_numpy(np.sin(ang).astype(np.float32)).cuda()
        s["qkv"] = torch.randn(s["nrow"], (nq + 2 * nkv) * HD, generator=gen, device="cuda")
        s["qn"], s["kn"] = (1 + 0.1 * torch.randn(2, HD, generator=gen, device="cuda")).unbind()
        s["q_out"] = torch.zeros(s["nrow"], nq, HD, device="cuda")
        return s
    s["pk"], s["pv"] = _cache(gen, nkv, case["prefix"] + 3)
    s["plen"] = _i32([case["prefix"]])
    s["q"] = _queries(gen, s["nrow"], nkv, group, s["pk"][:, :case["prefix"]])
    s["ctx"] = torch.zeros(s["nrow"], nq, HD, device="cuda")
    return s


# ---- the framework's calls -----------------------------------------------------------

_lib = None


def _hv():
    global _lib
    if _lib is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import hvdrv
        hvdrv.load()
        _lib = hvdrv
    return _lib


def _scratch(s, size, *args):
    """A program's workspace for a call, kept beside its inputs and zeroed once."""
    if "scratch" not in s:
        s["scratch"] = torch.zeros(max(size(*args), 16), dtype=torch.uint8, device="cuda")
    return s["scratch"].data_ptr()


def _run_own(s):
    hv = _hv()
    st = torch.cuda.current_stream().cuda_stream
    nkv, op = s["nkv"], s["op"]
    if op == "evict":
        ko, vo, mo, kept, left = s["out"]
        n, keep, nset = s["n"], s["keep"], s["nset"]
        scr = _scratch(s, hv.kv_evict_scratch, nkv, n, nset)
        hv.kv_evict(s["k"].data_ptr(), s["v"].data_ptr(), nkv * n * HD, s["mass"].data_ptr(), n,
                    s["len"].data_ptr(), 0, ko.data_ptr(), vo.data_ptr(), nkv * keep * HD,
                    mo.data_ptr(), keep, left.data_ptr(), kept.data_ptr(), keep, keep,
                    s["recent"], nkv, HD, nset, scr, st)
        return ko, vo, mo, kept, left
    group = s["group"]
    nq = nkv * group
    if op == "mass":
        ctx, mo = s["out"]
        scr = _scratch(s, hv.attn_mass_scratch, nq, group, s["cap"], s["ntok"])
        if s["ntok"] == 1:
            hv.attn_decode_mass(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                                ctx.data_ptr(), s["mass"].data_ptr(), mo.data_ptr(),
                                s["scale"].data_ptr(), s["pos"].data_ptr(), nq, HD, group,
                                s["cap"], scr, st)
        else:
            hv.attn_rows_mass(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                              ctx.data_ptr(), s["mass"].data_ptr(), mo.data_ptr(),
                              s["scale"].data_ptr(), s["pos0"], nq, HD, group, s["cap"],
                              s["ntok"], scr, st)
        return ctx, mo
    if op == "tails":
        hv.qk_shared(s["qkv"].data_ptr(), s["qn"].data_ptr(), s["kn"].data_ptr(),
                     s["cos"].data_ptr(), s["sin"].data_ptr(), s["cap"], s["base"].data_ptr(),
                     s["row0"].data_ptr(), s["tlen"].data_ptr(), s["q_out"].data_ptr(),
                     s["tk"].data_ptr(), s["tv"].data_ptr(), nq, nkv, HD, s["tcap"], EPS,
                     s["nseq"], s["nrow"], st)
        return s["q_out"], s["tk"], s["tv"]
    scr = _scratch(s, hv.attn_shared_scratch, nq, group, s["prefix"] + 3, s["tcap"], s["nseq"],
                   s["nrow"])
    hv.attn_shared(s["q"].data_ptr(), s["pk"].data_ptr(), s["pv"].data_ptr(), s["prefix"] + 3,
                   s["plen"].data_ptr(), s["tk"].data_ptr(), s["tv"].data_ptr(), s["tcap"],
                   s["row0"].data_ptr(), s["tlen"].data_ptr(), s["ctx"].data_ptr(),
                   s["scale"].data_ptr(), nq, HD, group, s["nseq"], s["nrow"], scr, st)
    return s["ctx"]


# ---- the plain forms -----------------------------------------------------------------

def _plain_evict(s):
    n, keep, recent = s["n"], s["keep"], s["recent"]
    if keep >= n:
        idx = torch.arange(n, device="cuda").expand(s["nset"], s["nkv"], n)
    else:
        old = n - recent
        top = torch.sort(s["mass"][..., :old], dim=-1, descending=True, stable=True).indices
        late = torch.arange(old, n, device="cuda").expand(s["nset"], s["nkv"], recent)
        idx = torch.cat([torch.sort(top[..., :keep - recent], dim=-1).values, late], -1)
    rows = idx[..., None].expand(*idx.shape, HD)
    return (torch.gather(s["k"], 2, rows), torch.gather(s["v"], 2, rows),
            torch.gather(s["mass"], 2, idx), idx.to(torch.int32),
            torch.full_like(s["len"], idx.shape[-1]))


def _plain_mass(s):
    nkv, group, ntok, pos0 = s["nkv"], s["group"], s["ntok"], s["pos0"]
    n = pos0 + ntok
    q = s["q"].reshape(ntok, nkv, group, HD).permute(1, 0, 2, 3).reshape(nkv, ntok * group, HD)
    hidden = (torch.arange(n, device="cuda")[None, :]
              > (pos0 + torch.arange(ntok, device="cuda").repeat_interleave(group))[:, None])
    ctx = torch.empty(nkv, ntok * group, HD, device="cuda")
    mass = torch.zeros(nkv, s["cap"], device="cuda")
    some = max(1, 2 ** 26 // (ntok * group * n))        # heads at a time: the scores stay small
    for h in range(0, nkv, some):
        at = slice(h, h + some)
        x = (q[at] @ s["k"][at, :n].float().transpose(1, 2)) * s["scale"]
        x = x.masked_fill(hidden, -math.inf)
        w = torch.exp(x - x.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        ctx[at] = w @ s["v"][at, :n].float()
        mass[at, :n] = s["mass"][at, :n] + w.sum(1)
    ctx = ctx.reshape(nkv, ntok, group, HD).permute(1, 0, 2, 3)
    return ctx.reshape(ntok, nkv * group, HD).contiguous(), mass


def _plain_tails(s):
    nkv, nq = s["nkv"], s["nkv"] * s["group"]
    x = s["qkv"].reshape(s["nrow"], nq + 2 * nkv, HD)
    pos = s["base"].long() + s["slot"]
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(y, w):
        y = w * (y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS))
        lo, hi = y[..., :HD // 2], y[..., HD // 2:]
        return torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)

    s["tk"][s["seq"], :, s["slot"]] = turned(x[:, nq:nq + nkv], s["kn"]).half()
    s["tv"][s["seq"], :, s["slot"]] = x[:, nq + nkv:].half()
    return turned(x[:, :nq], s["qn"]), s["tk"], s["tv"]


def _plain_shared(s):
    nkv, group, nrow, npre = s["nkv"], s["group"], s["nrow"], s["prefix"]
    nseq, tcap, most = s["nseq"], s["tcap"], max(s["row_list"])
    q = s["q"].reshape(nrow, nkv, group, HD)
    flat = q.permute(1, 0, 2, 3).reshape(nkv, nrow * group, HD)
    xp = (flat @ s["pk"][:, :npre].float().transpose(1, 2)).reshape(nkv, nrow, group, npre)
    # the sequences' rows side by side, each against its own tail
    at = s["row0"][:-1].long()[s["seq"]]
    lane = torch.arange(nrow, device="cuda") - at
    qs = torch.zeros(nseq, nkv, most, group, HD, device="cuda")
    qs[s["seq"], :, lane] = q
    xt = qs.reshape(nseq, nkv, most * group, HD) @ s["tk"].float().transpose(2, 3)
    xt = xt.reshape(nseq, nkv, most, group, tcap)[s["seq"], :, lane].permute(1, 0, 2, 3)
    out = torch.arange(tcap, device="cuda")[None, :] > s["slot"][:, None]
    xt = xt.masked_fill(out[None, :, None], -math.inf)
    x = torch.cat([xp, xt], -1) * s["scale"]
    w = torch.exp(x - x.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = (w[..., :npre].reshape(nkv, nrow * group, npre) @ s["pv"][:, :npre].float())
    o = o.reshape(nkv, nrow, group, HD).permute(1, 0, 2, 3)
    wt = torch.zeros(nseq, nkv, most, group, tcap, device="cuda")
    wt[s["seq"], :, lane] = w[..., npre:].permute(1, 0, 2, 3)
    ot = wt.reshape(nseq, nkv, most * group, tcap) @ s["tv"].float()
    ot = ot.reshape(nseq, nkv, most, group, HD)[s["seq"], :, lane]
    return (o + ot).reshape(nrow, nkv * group, HD)


_PLAIN = {"evict": _plain_evict, "mass": _plain_mass, "tails": _plain_tails,
          "shared": _plain_shared}


def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------

def _exact_evict(s):
    n, keep, recent = s["n"], s["keep"], s["recent"]
    mass = s["mass"].cpu().numpy()
    kept = np.empty((s["nset"], s["nkv"], keep), np.int32)
    for i in range(s["nset"]):
        for h in range(s["nkv"]):
            old = mass[i, h, :n - recent]
            best = np.lexsort((np.arange(old.size), -old))[:keep - recent]
            kept[i, h] = np.concatenate([np.sort(best), np.arange(n - recent, n)])
    idx = torch.from_numpy(kept).long().cuda()
    i, h = (torch.arange(m, device="cuda") for m in idx.shape[:2])
    at = (i[:, None, None], h[None, :, None], idx)
    return (s["k"][at], s["v"][at], s["mass"][at].double(), idx.to(torch.int32),
            torch.full_like(s["len"], keep))


def _attend(q, k, v, seen, scale):
    """One head: q [m, 128] over k, v [n, 128], row r over the positions where seen [m, n]; the
    context and the weights."""
    x = (q @ k.T) * scale
    x[~seen] = -math.inf
    w = torch.softmax(x, -1)
    return w @ v, w


def _exact_mass(s):
    nkv, group, ntok, pos0 = s["nkv"], s["group"], s["ntok"], s["pos0"]
    n = pos0 + ntok
    q, scale = s["q"].double().reshape(ntok, nkv, group, HD), s["scale"].double()
    ctx = torch.empty(ntok, nkv, group, HD, dtype=torch.float64, device="cuda")
    mass = torch.zeros(nkv, s["cap"], dtype=torch.float64, device="cuda")
    mass[:, :n] = s["mass"].double()[:, :n]
    seen = (torch.arange(n, device="cuda")[None, :]
            <= pos0 + torch.arange(ntok, device="cuda")[:, None])
    for h in range(nkv):
        k, v = s["k"][h, :n].double(), s["v"][h, :n].double()
        for g in range(group):
            ctx[:, h, g], w = _attend(q[:, h, g], k, v, seen, scale)
            mass[h, :n] += w.sum(0)
    return ctx.reshape(ntok, nkv * group, HD), mass


def _exact_tails(s):
    nkv, nq = s["nkv"], s["nkv"] * s["group"]
    x = s["qkv"].double().reshape(s["nrow"], nq + 2 * nkv, HD)
    pos = s["prefix"] + s["slot"]
    turn = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]

    def heads(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(y[..., :HD // 2], y[..., HD // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    tk, tv = s["tk"].double(), s["tv"].double()
    tk[s["seq"], :, s["slot"]] = heads(x[:, nq:nq + nkv], s["kn"])
    tv[s["seq"], :, s["slot"]] = x[:, nq + nkv:]
    return heads(x[:, :nq], s["qn"]), tk, tv


def _exact_shared(s):
    nkv, group, npre = s["nkv"], s["group"], s["prefix"]
    q, scale = s["q"].double().reshape(s["nrow"], nkv, group, HD), s["scale"].double()
    ctx = torch.empty_like(q)
    for h in range(nkv):
        pk, pv = s["pk"][h, :npre].double(), s["pv"][h, :npre].double()
        r0 = 0
        for i, (r, t) in enumerate(zip(s["row_list"], s["tail_list"])):
            k = torch.cat([pk, s["tk"][i, h, :t].double()])
            v = torch.cat([pv, s["tv"][i, h, :t].double()])
            see = npre + t - r + torch.arange(r, device="cuda").repeat_interleave(group)
            seen = torch.arange(npre + t, device="cuda")[None, :] <= see[:, None]
            o, _ = _attend(q[r0:r0 + r, h].reshape(r * group, HD), k, v, seen, scale)
            ctx[r0:r0 + r, h] = o.reshape(r, group, HD)
            r0 += r
    return ctx.reshape(s["nrow"], nkv * group, HD)


_EXACT = {"evict": _exact_evict, "mass": _exact_mass, "tails": _exact_tails,
          "shared": _exact_shared}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
