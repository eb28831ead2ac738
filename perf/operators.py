"""What is measured of the 8-bit KV cache and of scoring: the cases, the operators' plain
forms and their values in 64 bits.

Four operators, each through the entry points of hvdrv.py that a program calls:

  kv      rows of K and V quantised as they are written (kv_append_q8 for one token at a
          device-resident position, kv_rows_q8 for a run of rows), then every position of
          the blocks they touch read back as f32 (kv_read_q8)
  decode  attention of one query token over the cache (attn_decode_q8)
  rows    causal attention of a run of query tokens over the cache (attn_rows_q8)
  score   log probabilities of given tokens, with the entropy of each distribution and its
          most likely alternatives (logprob_rows)

The cache holds, for every kv head and every block of 32 positions, int8 codes of the
block's 32 x 128 K values and one f32 scale, and the same for V:

  s = f32(max|x| / 127), 1 where that is 0;  c = trunc(f32(x / s) + (x < 0 ? -0.5 : 0.5)),
  clipped to +-127;  the value read is f32(c s).

The block that is still open (fewer than 32 rows written) is kept in f32 and is quantised
once, when its last row arrives.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False          # set by the tools: True makes the calls of the framework's kernels

BLK, HD = 32, 128
_PKG = str(Path(__file__).resolve().parent.parent / "hive-limited_b200")


def listed():
    return [
        # a decode step's append: one row per kv head, the one that completes a block
        dict(name="kv-append-1", op="kv", nkv=8, pos0=4223, ntok=1),
        # one run of the batched prefill (256 tokens of a 4096-token prompt)
        dict(name="kv-run-256", op="kv", nkv=8, pos0=3840, ntok=256),
        # a whole long prompt at once, ending inside a block
        dict(name="kv-prompt-16377", op="kv", nkv=8, pos0=0, ntok=16377),
        # the first decode steps after a short prompt: 16 q heads over 8 kv heads
        dict(name="decode-45", op="decode", nkv=8, group=2, n=45),
        # decode inside the 4096 + 256 token workload, 32 q heads over 8 kv heads
        dict(name="decode-4225", op="decode", nkv=8, group=4, n=4225),
        # 64 q heads over 8 kv heads at a long context
        dict(name="decode-39999", op="decode", nkv=8, group=8, n=39999),
        # the longest cache of the range
        dict(name="decode-131072", op="decode", nkv=8, group=4, n=131072),
        # the second run of a 300-token prompt, 16 q heads over 8 kv heads: ragged
        dict(name="rows-44-at-256", op="rows", nkv=8, group=2, pos0=256, ntok=44),
        # the last run of a 4096-token prompt, 32 q heads over 8 kv heads
        dict(name="rows-256-at-3840", op="rows", nkv=8, group=4, pos0=3840, ntok=256),
        # a run deep in a 16k prompt, 64 q heads over 8 kv heads
        dict(name="rows-256-at-16128", op="rows", nkv=8, group=8, pos0=16128, ntok=256),
        # one step's logits: the token's log probability and 20 alternatives
        dict(name="score-1-top20", op="score", rows=1, vocab=151936, top=20),
        # a prompt run scored at every position, 5 alternatives each
        dict(name="score-256-top5", op="score", rows=256, vocab=151936, top=5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["kv", "decode", "decode", "rows", "rows", "score"])
    if op == "kv":
        ntok = 1 if rng.random() < 0.3 else _log(rng, 2, 16000)
        return dict(op=op, nkv=rng.choice([1, 2, 4, 8]), pos0=rng.randrange(0, 5000), ntok=ntok)
    if op == "decode":
        return dict(op=op, nkv=rng.choice([1, 2, 4, 8]), group=rng.randint(1, 8),
                    n=_log(rng, 1, 65536))
    if op == "rows":
        return dict(op=op, nkv=rng.choice([2, 4, 8]), group=rng.choice([1, 2, 4, 5, 8]),
                    pos0=_log(rng, 1, 16000) - 1, ntok=_log(rng, 1, 256))
    return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 151936),
                top=rng.randint(0, 20))


def work(case):
    """Each input read once and each output written once: codes are 1 byte, scales 4 per
    block of 32 positions, open rows, queries, contexts and logits f32."""
    if case["op"] == "kv":
        first = case["pos0"] // BLK * BLK
        new, back = case["ntok"], case["pos0"] + case["ntok"] - first
        per = 2 * case["nkv"] * HD
        return {"bytes": per * (4 * new + back + back + 4 * back), "flops": per * 5 * back}
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 8 * case["rows"] * (1 + case["top"]), "flops": 6 * n}
    n = case["n"] if case["op"] == "decode" else case["pos0"] + case["ntok"]
    ntok = case.get("ntok", 1)
    nq = case["nkv"] * case["group"]
    closed = n // BLK * BLK
    cache = 2 * case["nkv"] * (closed * HD + closed // BLK * 4 + (n - closed) * HD * 4)
    seen = ntok * n - ntok * (ntok - 1) // 2                 # (query, position) pairs
    return {"bytes": cache + 2 * ntok * nq * HD * 4, "flops": 4 * nq * HD * seen}


# ---- the cache's arrangement ---------------------------------------------------------

def _quantise(x):
    """Blocks x [..., 32, 128] f32 -> codes int8, scales f32 [...]."""
    s = x.abs().amax((-2, -1))
    s = s / torch.full_like(s, 127.0)         # a true division: by a number it is a product
    s = torch.where(s == 0, torch.ones_like(s), s)
    t = x / s[..., None, None]
    c = torch.trunc(t + torch.where(x < 0, -0.5, 0.5)).clamp(-127, 127)
    return c.to(torch.int8), s


def _cache_bytes(nkv, cap):
    nblk = -(-cap // BLK)
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    codes, scales = nkv * nblk * 2 * BLK * HD, up(nkv * nblk * 8)
    tail, state = nkv * 2 * BLK * HD * 4, up(nkv * 8)
    return nblk, (codes, codes + scales, codes + scales + tail, codes + scales + tail + state)


def _arranged(kc, vc, ks, vs, tail, n, cap):
    """The buffer a program's cache is, holding n positions: kc, vc codes [nkv, nb, 32, 128]
    and ks, vs scales [nkv, nb] of the complete blocks, tail [nkv, 2, 32, 128] the rows of the
    last block in f32. include/hive_b200.h documents the arrangement."""
    nkv, nb = kc.shape[:2]
    nblk, (o_s, o_t, o_l, total) = _cache_bytes(nkv, cap)
    buf = torch.zeros(total, dtype=torch.uint8, device="cuda")
    codes = buf[:o_s].view(nkv, nblk, 2, BLK * HD)
    kp = kc.view(nkv, nb, 4, 8, 2, 4, 4, 4).permute(0, 1, 2, 4, 3, 6, 5, 7)
    vp = vc.view(nkv, nb, 2, 2, 4, 2, 8, 2, 8).permute(0, 1, 6, 8, 4, 7, 2, 3, 5)
    codes[:, :nb, 0] = (kp.reshape(nkv, nb, BLK * HD).to(torch.int16) + 128).to(torch.uint8)
    codes[:, :nb, 1] = (vp.reshape(nkv, nb, BLK * HD).to(torch.int16) + 128).to(torch.uint8)
    sc = buf[o_s:o_s + nkv * nblk * 8].view(torch.float32).view(nkv, nblk, 2)
    sc[:, :nb, 0], sc[:, :nb, 1] = ks, vs
    buf[o_t:o_l].view(torch.float32).view(nkv, 2, BLK, HD).copy_(tail)
    buf[o_l:o_l + nkv * 8].view(torch.int32).fill_(n)
    return buf


def _history(gen, nkv, n):
    """K and V rows [nkv, n, 128] as a model writes them: keys of unit scale after their norm
    with some dimensions larger, values a little smaller."""
    k = torch.randn(nkv, n, HD, generator=gen, device="cuda")
    k *= torch.exp(0.3 * torch.randn(nkv, 1, HD, generator=gen, device="cuda"))
    v = 0.7 * torch.randn(nkv, n, HD, generator=gen, device="cuda") + 0.1
    return k, v


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "score":
        r, v = case["rows"], case["vocab"]
        s["logits"] = 2.5 * torch.randn(r, v, generator=gen, device="cuda")
        s["logits"][:, ::997] += 6.0 * torch.rand(r, 1, generator=gen, device="cuda")
        s["tok"] = torch.randint(0, v, (r,), generator=gen, device="cuda", dtype=torch.int32)
        s["out"] = [torch.zeros(r, device="cuda"), torch.zeros(r, device="cuda"),
                    torch.zeros(r, case["top"], dtype=torch.int32, device="cuda"),
                    torch.zeros(r, case["top"], device="cuda")]
        return s
    nkv = case["nkv"]
    if case["op"] == "kv":
        first, pos0, ntok = case["pos0"] // BLK * BLK, case["pos0"], case["ntok"]
        k, v = _history(gen, nkv, pos0 - first + ntok)
        tail = torch.zeros(nkv, 2, BLK, HD, device="cuda")
        tail[:, 0, :pos0 - first], tail[:, 1, :pos0 - first] = k[:, :pos0 - first], v[:, :pos0 - first]
        s["tail"] = tail
        s["k"] = k[:, pos0 - first:].transpose(0, 1).contiguous()      # [ntok, nkv, 128]
        s["v"] = v[:, pos0 - first:].transpose(0, 1).contiguous()
        s["cap"] = pos0 + ntok
        none = torch.zeros(nkv, 0, BLK, HD, dtype=torch.int8, device="cuda")
        flat = torch.zeros(nkv, 0, device="cuda")
        s["kv"] = _arranged(none, none, flat, flat, tail, pos0, s["cap"])
        s["pos"] = torch.tensor([pos0], dtype=torch.int32, device="cuda")
        s["out"] = [torch.zeros(pos0 - first + ntok, nkv, HD, device="cuda") for _ in range(2)]
        return s
    n = case["n"] if case["op"] == "decode" else case["pos0"] + case["ntok"]
    ntok = case.get("ntok", 1)
    nq = nkv * case["group"]
    k, v = _history(gen, nkv, n)
    q = torch.randn(ntok, nkv, case["group"], HD, generator=gen, device="cuda")
    # some positions that the query looks for, so that the weights are not flat
    at = torch.randint(0, max(1, n - ntok + 1), (nkv, 4), generator=gen, device="cuda")
    look = torch.gather(k, 1, at[..., None].expand(nkv, 4, HD)).mean(1)
    s["q"] = (q + 0.8 * look[None, :, None]).reshape(ntok, nq, HD).contiguous()
    closed = n // BLK * BLK
    blocks = lambda x: x[:, :closed].reshape(nkv, closed // BLK, BLK, HD)  # noqa: E731
    (s["kc"], s["ks"]), (s["vc"], s["vs"]) = _quantise_all(blocks(k)), _quantise_all(blocks(v))
    s["kt"], s["vt"] = k[:, closed:].contiguous(), v[:, closed:].contiguous()
    tail = torch.zeros(nkv, 2, BLK, HD, device="cuda")
    last = (n - 1) // BLK * BLK
    tail[:, 0, :n - last], tail[:, 1, :n - last] = k[:, last:], v[:, last:]
    s["cap"] = n
    s["kv"] = _arranged(s["kc"], s["vc"], s["ks"], s["vs"], tail, n, n)
    s["scale"] = torch.tensor([1.0 / math.sqrt(HD)], device="cuda")
    s["pos"] = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    s["ctx"] = torch.zeros(ntok, nq, HD, device="cuda")
    return s


def _quantise_all(x):
    """_quantise in slices of one head, to keep the temporaries small."""
    c = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(x.shape[:2], device=x.device)
    if x.shape[1]:
        for h in range(x.shape[0]):
            c[h], s[h] = _quantise(x[h])
    return c, s


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


def _scratch(s, nbytes):
    """A program's workspace for a call, kept beside its inputs and zeroed once."""
    if "scratch" not in s:
        s["scratch"] = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    return s["scratch"].data_ptr()


def _run_own(s):
    hv = _hv()
    st = torch.cuda.current_stream().cuda_stream
    if s["op"] == "kv":
        nkv, cap, pos0, ntok, kv = s["nkv"], s["cap"], s["pos0"], s["ntok"], s["kv"].data_ptr()
        if ntok == 1:
            hv.kv_append_q8(s["k"].data_ptr(), s["v"].data_ptr(), kv, s["pos"].data_ptr(), nkv,
                            HD, cap, st)
        else:
            hv.kv_rows_q8(s["k"].data_ptr(), s["v"].data_ptr(), nkv * HD, kv, pos0, nkv, HD, cap,
                          ntok, st)
        first = pos0 // BLK * BLK
        ko, vo = s["out"]
        hv.kv_read_q8(kv, ko.data_ptr(), vo.data_ptr(), first, nkv, HD, cap, pos0 + ntok - first,
                      st)
        return ko, vo
    if s["op"] == "score":
        lp, ent, ids, alt = s["out"]
        r, v, top = s["rows"], s["vocab"], s["top"]
        scr = s.get("scratch_ptr") or _scratch(s, hv.logprob_scratch(r, v, top))
        s["scratch_ptr"] = scr
        hv.logprob_rows(s["logits"].data_ptr(), v, r, v, s["tok"].data_ptr(), top, lp.data_ptr(),
                        ent.data_ptr(), ids.data_ptr() if top else 0, alt.data_ptr() if top else 0,
                        scr, st)
        return lp, ent, ids, alt
    nkv, group, cap = s["nkv"], s["group"], s["cap"]
    ntok = s.get("ntok", 1)
    scr = s.get("scratch_ptr") or _scratch(s, hv.attn_q8_scratch(nkv * group, group, cap, ntok))
    s["scratch_ptr"] = scr
    if s["op"] == "decode":
        hv.attn_decode_q8(s["q"].data_ptr(), s["kv"].data_ptr(), s["ctx"].data_ptr(),
                          s["scale"].data_ptr(), s["pos"].data_ptr(), nkv * group, HD, group, cap,
                          scr, st)
    else:
        hv.attn_rows_q8(s["q"].data_ptr(), s["kv"].data_ptr(), s["ctx"].data_ptr(),
                        s["scale"].data_ptr(), s["pos0"], nkv * group, HD, group, cap, ntok, scr,
                        st)
    return s["ctx"]


# ---- the plain forms -----------------------------------------------------------------

def _plain_kv(s):
    nkv, pos0, ntok = s["nkv"], s["pos0"], s["ntok"]
    old = pos0 % BLK
    n = old + ntok
    closed = n // BLK * BLK
    out = []
    for x, which in ((s["k"], 0), (s["v"], 1)):
        rows = torch.cat([s["tail"][:, which, :old], x.transpose(0, 1)], 1)   # [nkv, n, 128]
        c, sc = _quantise(rows[:, :closed].reshape(nkv, closed // BLK, BLK, HD)) if closed else (
            rows[:, :0].reshape(nkv, 0, BLK, HD), rows.new_zeros(nkv, 0))
        back = (c.float() * sc[..., None, None]).reshape(nkv, closed, HD)
        out.append(torch.cat([back, rows[:, closed:]], 1).transpose(0, 1).contiguous())
    return tuple(out)


def _plain_attention(s):
    nkv, group = s["nkv"], s["group"]
    ntok = s.get("ntok", 1)
    k = torch.cat([(s["kc"].float() * s["ks"][..., None, None]).flatten(1, 2), s["kt"]], 1)
    v = torch.cat([(s["vc"].float() * s["vs"][..., None, None]).flatten(1, 2), s["vt"]], 1)
    n = k.shape[1]
    q = s["q"].reshape(ntok, nkv, group, HD).permute(1, 0, 2, 3).reshape(nkv, ntok * group, HD)
    x = (q @ k.transpose(1, 2)) * s["scale"]
    if ntok > 1:
        last = n - ntok + torch.arange(ntok, device="cuda").repeat_interleave(group)
        x = x.masked_fill(torch.arange(n, device="cuda")[None, :] > last[:, None], -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    o = (w @ v) / w.sum(-1, keepdim=True)
    o = o.reshape(nkv, ntok, group, HD).permute(1, 0, 2, 3)
    return o.reshape(ntok, nkv * group, HD).contiguous()


def _plain_score(s):
    x, top = s["logits"], s["top"]
    at = torch.arange(s["rows"], device="cuda")
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1)
    lse = torch.log(total)
    lp = z[at, s["tok"].long()] - lse
    ent = lse - (z * e).sum(-1) / total
    # order by value, ties to the lower id: the f32 bits as an ordered integer, then ~id
    u = torch.where(x == 0, torch.zeros_like(x), x).view(torch.int32).long()
    u = torch.where(u < 0, -(u & 0x7FFFFFFF) - 1, u)
    key = (u << 32) | (0xFFFFFFFF - torch.arange(s["vocab"], device="cuda"))
    ids = (0xFFFFFFFF - (torch.topk(key, top, dim=-1).values & 0xFFFFFFFF)).to(torch.int32)
    alt = torch.gather(z, 1, ids.long()) - lse[:, None]
    return lp, ent, ids, alt


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "kv":
        return _plain_kv(state)
    return _plain_score(state) if state["op"] == "score" else _plain_attention(state)


# ---- the definition in 64 bits -------------------------------------------------------

def _exact_kv(s):
    """Row by row of blocks in numpy: the scale and the code are f32 by definition, the value
    they stand for is their product."""
    f = np.float32
    old, ntok, nkv = s["pos0"] % BLK, s["ntok"], s["nkv"]
    outs = []
    for name, which in (("k", 0), ("v", 1)):
        new = s[name].cpu().numpy()
        rows = np.empty((old + ntok, nkv, HD), f)
        rows[:old] = s["tail"][:, which, :old].cpu().numpy().swapaxes(0, 1)
        rows[old:] = new
        out = rows.astype(np.float64)
        for b in range(0, (old + ntok) // BLK * BLK, BLK):
            x = rows[b:b + BLK]
            sc = (np.abs(x).max(axis=(0, 2), keepdims=True) / f(127)).astype(f)
            sc[sc == 0] = 1
            q = (x / sc).astype(f)
            c = np.fix((q + np.where(x < 0, f(-0.5), f(0.5))).astype(f))
            out[b:b + BLK] = np.clip(c, -127, 127).astype(np.float64) * sc.astype(np.float64)
        outs.append(torch.from_numpy(out))
    return tuple(outs)


def _exact_attention(s):
    nkv, group = s["nkv"], s["group"]
    ntok, n = s.get("ntok", 1), s["cap"]
    q = s["q"].double().reshape(ntok, nkv, group, HD)
    out = torch.empty(ntok, nkv, group, HD, dtype=torch.float64, device="cuda")
    pos = torch.arange(n, device="cuda")
    for h in range(nkv):
        deq = [torch.cat(((c[h].double() * sc[h].double()[:, None, None]).flatten(0, 1),
                          t[h].double())) for c, sc, t in ((s["kc"], s["ks"], s["kt"]),
                                                           (s["vc"], s["vs"], s["vt"]))]
        for g in range(group):
            x = (q[:, h, g] @ deq[0].T) * s["scale"].double()
            if ntok > 1:
                hidden = pos[None, :] > (n - ntok + torch.arange(ntok, device="cuda"))[:, None]
                x[hidden] = -math.inf
            out[:, h, g] = torch.softmax(x, -1) @ deq[1]
    return out.reshape(ntok, nkv * group, HD)


def _exact_score(s):
    x = s["logits"].double()
    lps = torch.log_softmax(x, -1)
    p = torch.exp(lps)
    lp = lps.gather(1, s["tok"].long()[:, None])[:, 0]
    ent = -(p * lps).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    return lp, ent, order.to(torch.int32), lps.gather(1, order)


def exact(case, seed):
    s = prepare(case, seed)
    return {"kv": _exact_kv, "score": _exact_score}.get(case["op"], _exact_attention)(s)
