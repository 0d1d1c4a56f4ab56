"""Timed cases of the 8-bit paged K/V operators: what their users run, through the public entry points.

Three kinds of case.

- ``append``: the fresh q, k and v rows of some sequences: q and k rotated (with or without the per-head norm), k and v
  quantised into the 8-bit pages (``cj_kv8_append``), and the 16-position blocks that this changed read back as the
  values they now stand for (``cj_kv8_read``).
- ``decode``: one layer's attention of one fresh token (or a few) for each sequence of a batch (``cj_kv8_attend``).
- ``chunk``: the same attention for prefill chunks: many rows a sequence, causal (``cj_kv8_attend``).

The cache. A page holds 64 positions of every kv head; a slot's pages stand in its row of the page table. K codes are
[page][kv head][64][hd] bytes, V codes [page][kv head][4 blocks][hd][16], a code the byte less 128; after the codes of a
plane come its scales, [page][kv head][4] floats, one power of two for each block of 16 positions of a head.

A segment is {slot, position, row, rows}: ``rows`` rows of q, k, v and out from ``row`` on are the slot's positions from
``position`` on. All inputs are made on the GPU from the seed alone.
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAGE, BLOCK = 64, 16
THETA = 500000.0
EPS = 1e-5
LOW, HIGH = -48, 63          # the scales' exponents

# query heads, kv heads, head size
SHAPES = {"tiny": (8, 2, 64), "dense": (32, 8, 128), "moe": (64, 8, 64)}


def listed():
    def case(name, kind, shape, seqs, count, rows, ragged=False, norm=False, window=0):
        return {"name": name, "kind": kind, "shape": shape, "seqs": seqs, "count": count, "rows": rows, "ragged": ragged,
                "norm": norm, "window": window}

    return [
        # the smallest call: one token of one short sequence of the tiny model
        case("append_tiny_1", "append", "tiny", 1, 101, 1),
        # a decode step of a batch: one token for each of 64 sequences of all lengths, most inside a block
        case("append_dense_64x1", "append", "dense", 64, 2048, 1, ragged=True),
        # a whole prefill chunk that begins inside a block
        case("append_dense_512", "append", "dense", 1, 1545, 512),
        # the ragged prompts of several requests at once, with the per-head norm
        case("append_moe_16x300", "append", "moe", 16, 300, 300, ragged=True, norm=True),
        # one token of one short sequence: latency alone
        case("decode_tiny_101", "decode", "tiny", 1, 101, 1),
        # one token at the 2049-position context, 8B shape: few heads, so the positions are split
        case("decode_dense_2049", "decode", "dense", 1, 2049, 1),
        # a serving batch of ragged lengths
        case("decode_dense_32x4096", "decode", "dense", 32, 4096, 1, ragged=True),
        # head size 64 with eight heads a kv head; three rows a sequence, as a verified draft has them
        case("decode_moe_16x4097_3", "decode", "moe", 16, 4097, 3),
        # the largest cache: long contexts, read once
        case("decode_dense_8x65500", "decode", "dense", 8, 65500, 1),
        # a prefill chunk behind a cached prefix
        case("chunk_dense_512_at_1545", "chunk", "dense", 1, 2057, 512),
        # the ragged prompts of several requests in layers with a 128-position window
        case("chunk_moe_16x300_w128", "chunk", "moe", 16, 300, 300, ragged=True, window=128),
        # the largest: four whole prompts
        case("chunk_dense_4x4096", "chunk", "dense", 4, 4096, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "chunk"))
    shape = rng.choice(("tiny", "dense", "dense", "moe"))
    c = {"kind": kind, "shape": shape, "ragged": rng.random() < 0.6, "norm": kind == "append" and rng.random() < 0.4,
         "window": rng.choice((128, 1000)) if kind != "append" and rng.random() < 0.25 else 0}
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        count = _log(rng, 16, min(65500, 400000 // seqs))
        rows = rng.choice((1, 1, 1, 2, 4))
    else:
        seqs = _log(rng, 1, 16)
        rows = _log(rng, 5, 4096 // seqs)
        most = min(8192, (1 << 25) // (seqs * rows) - rows)   # no more work than the largest listed case
        count = rows + (0 if rng.random() < 0.4 or most < 1 else _log(rng, 1, most))
        if kind == "append" and rng.random() < 0.4:
            seqs, rows = _log(rng, 1, 128), 1
    return {**c, "seqs": seqs, "count": max(count, rows), "rows": rows}


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """(cached positions before, rows) of each sequence."""
    rng = random.Random("%d %d %d" % (case["count"], case["seqs"], case["rows"]))
    out = []
    for i in range(case["seqs"]):
        rows, before = case["rows"], case["count"] - case["rows"]
        if case["ragged"] and i:   # the first is the longest
            if rows > 8:
                rows = rng.randint(max(1, rows // 3), rows)
            before = rng.randint(before // 4, before) if before else 0
        out.append((before, rows))
    return out


def _quantised(x, dims):
    """Codes and scales of the blocks whose values lie along `dims`."""
    top = x.abs().amax(dims, keepdim=True)
    e = torch.ceil(torch.log2(top / 127)).clamp(LOW, HIGH)
    scale = torch.exp2(e)
    scale = torch.where(top > 127 * scale, scale * 2, scale)
    return (x / scale).round().to(torch.int16), scale


def _inputs(case, seed):
    heads, kv, hd = SHAPES[case["shape"]]
    lens = _lengths(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    need = [(b + r + PAGE - 1) // PAGE for b, r in lens]
    pool, slots, per = sum(need) + 3, case["seqs"] + 2, max(need) + 1
    # a slot's pages as they came off the pool; entries past its length are none
    order = torch.randperm(pool, generator=g, device="cuda").cpu().numpy().astype(np.int32)
    slot = np.random.RandomState(int(seed) % (1 << 31)).permutation(slots)[:case["seqs"]]
    table, segs, at, row = np.full((slots, per), -1, np.int32), np.zeros((case["seqs"], 4), np.int32), 0, 0
    for i, (before, rows) in enumerate(lens):
        table[slot[i], :need[i]] = order[at:at + need[i]]
        segs[i] = (slot[i], before, row, rows)
        at, row = at + need[i], row + rows
    planes, scales = [], []
    for which in range(2):
        codes = torch.empty((pool, kv, PAGE, hd) if which == 0 else (pool, kv, 4, hd, BLOCK), dtype=torch.uint8, device="cuda")
        scale = torch.empty(pool, kv, 4, dtype=torch.float32, device="cuda")
        loud = 1 + 0.5 * torch.rand(kv, 1, 1, 1, generator=g, device="cuda")   # heads differ in size, as trained ones do
        for p in range(0, pool, 512):
            n = min(512, pool - p)
            x = torch.randn(n, kv, 4, BLOCK, hd, generator=g, device="cuda") * loud
            c, s = _quantised(x, (3, 4))
            c = (c + 128).to(torch.uint8)
            codes[p:p + n] = c.reshape(n, kv, PAGE, hd) if which == 0 else c.transpose(3, 4)
            scale[p:p + n] = s.reshape(n, kv, 4)
        planes.append(codes)
        scales.append(scale)
    s = {"k_codes": planes[0], "v_codes": planes[1], "k_scale": scales[0], "v_scale": scales[1],
         "table": torch.from_numpy(table).cuda(), "segs": torch.from_numpy(segs).cuda(), "total": row}
    if case["kind"] == "append":
        # the rows of a fused projection: q, k and v of a row next to one another
        s["qkv"] = torch.randn(row, (heads + 2 * kv) * hd, generator=g, device="cuda")
        s["qw"] = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
        s["kw"] = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
        ctx = max(b + r for b, r in lens)
        inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        ang = torch.arange(ctx, dtype=torch.float64, device="cuda")[:, None] * inv
        s["rope"] = torch.stack((ang.cos(), ang.sin()), -1).float()   # [position][hd/2](cos, sin)
        # the blocks that the rows reach, whole, for the read: a segment from the first one's start
        back, at = segs.copy(), 0
        for i, (before, rows) in enumerate(lens):
            first = before // BLOCK * BLOCK
            back[i, 1:] = (first, at, before + rows - first)
            at += before + rows - first
        s["back"], s["back_total"] = torch.from_numpy(back).cuda(), at
    else:
        s["q"] = torch.randn(row, heads * hd, generator=g, device="cuda") * 1.5
    return s


# ------------------------------------------------------- the framework's side

def _package():
    name = "cajeta_llm_amd"
    if name not in sys.modules:
        d = os.path.join(ROOT, "cajeta-llm_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        m = importlib.util.module_from_spec(spec)
        sys.modules[name] = m
        spec.loader.exec_module(m)
        m.native.init(0)
        try:   # the registry's lookup of an optional kernel leaves the runtime's last error set; torch would report it
            torch.zeros(1, device="cuda")
        except RuntimeError:
            pass
    return sys.modules[name]


class _View:
    """A device buffer's memory, as torch takes it."""

    def __init__(self, buf, shape, dtype):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": dtype, "data": (buf.h, False), "version": 2}


def _view(buf, shape, dtype="<f4"):
    t = torch.as_tensor(_View(buf, shape, dtype), device="cuda")
    t._held = buf
    return t


def _buffer(pkg, *parts):
    """A device buffer of the framework that holds the tensors one after the other."""
    flat = [t.contiguous().view(torch.uint8).reshape(-1) for t in parts]
    buf = pkg.Buffer(max(16, sum(f.numel() for f in flat)))
    at, all_ = 0, _view(buf, (buf.nbytes,), "|u1")
    for f in flat:
        all_[at:at + f.numel()].copy_(f)
        at += f.numel()
    torch.cuda.synchronize()
    return buf


def prepare(case, seed):
    s = _inputs(case, seed)
    heads, kv, hd = SHAPES[case["shape"]]
    s["case"], s["shape"] = case, (heads, kv, hd)
    if not own:
        return s
    pkg = _package()
    L = pkg.native.lib()
    slots, per = s["table"].shape
    pool, total, seqs = s["k_codes"].shape[0], s["total"], case["seqs"]
    t = {"case": case, "shape": (heads, kv, hd), "L": L, "check": pkg.native.check, "pool": pool, "slots": slots, "per": per,
         "total": total, "kp": _buffer(pkg, s["k_codes"], s["k_scale"]), "vp": _buffer(pkg, s["v_codes"], s["v_scale"]),
         "table": _buffer(pkg, s["table"]), "segs": _buffer(pkg, s["segs"])}
    if case["kind"] == "append":
        t.update(qkv=_buffer(pkg, s["qkv"]), qw=_buffer(pkg, s["qw"]), kw=_buffer(pkg, s["kw"]), rope=_buffer(pkg, s["rope"]),
                 ctx=s["rope"].shape[0], back=_buffer(pkg, s["back"]), back_total=s["back_total"],
                 q=pkg.Buffer(total * heads * hd * 4), ko=pkg.Buffer(s["back_total"] * kv * hd * 4),
                 vo=pkg.Buffer(s["back_total"] * kv * hd * 4))
        t["out"] = {"q": _view(t["q"], (total, heads * hd)), "k": _view(t["ko"], (s["back_total"], kv * hd)),
                    "v": _view(t["vo"], (s["back_total"], kv * hd))}
    else:
        t.update(q=_buffer(pkg, s["q"]), y=pkg.Buffer(total * heads * hd * 4))
        need = L.cj_kv8_attend_bytes(seqs, case["rows"], case["count"], heads, kv, hd, case["window"])
        t["part"] = pkg.Buffer(max(16, need))
        t["out"] = _view(t["y"], (total, heads * hd))
    return t


def _run_own(s):
    L, check, c = s["L"], s["check"], s["case"]
    heads, kv, hd = s["shape"]
    if c["kind"] == "append":
        wide, at = (heads + 2 * kv) * hd, s["qkv"].h
        check(L.cj_kv8_append(s["q"].h, at, at + 4 * heads * hd, at + 4 * (heads + kv) * hd, s["kp"].h, s["vp"].h, s["qw"].h,
                              s["kw"].h, s["rope"].h, s["table"].h, s["segs"].h, c["seqs"], c["rows"], s["total"], s["ctx"],
                              s["pool"], s["slots"], s["per"], heads, kv, hd, heads * hd, wide, wide, int(c["norm"]),
                              ctypes.c_float(EPS), 0, 0), "append")
        check(L.cj_kv8_read(s["ko"].h, s["vo"].h, s["kp"].h, s["vp"].h, s["table"].h, s["back"].h, c["seqs"],
                            c["rows"] + BLOCK - 1, s["back_total"], s["pool"], s["slots"], s["per"], kv, hd, kv * hd, 0), "read")
    else:
        check(L.cj_kv8_attend(s["y"].h, s["q"].h, s["kp"].h, s["vp"].h, s["table"].h, s["segs"].h, s["part"].h, c["seqs"],
                              c["rows"], s["total"], c["count"], s["pool"], s["slots"], s["per"], heads, kv, hd, heads * hd,
                              heads * hd, c["window"], ctypes.c_float(1 / math.sqrt(hd)), 0), "attend")
    return s["out"]


# --------------------------------------------------------- the plain forms

def _turned(x, cs):
    """x [..., hd] with the pairs (d, d + hd/2) rotated by cs [..., hd/2, 2]."""
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half], x[..., half:], cs[..., 0], cs[..., 1]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def _normed(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _run_append(s):
    heads, kv, hd = s["shape"]
    c, segs, table = s["case"], s["segs"].long(), s["table"].long()
    slot, pos, row, rows = segs.unbind(1)
    # which row is which position, and the rotated rows: in 64 bits, as codes next to a border need
    of = torch.repeat_interleave(torch.arange(len(segs), device="cuda"), rows, output_size=s["total"])
    at = pos[of] + torch.arange(s["total"], device="cuda") - row[of]
    x = s["qkv"].double().reshape(s["total"], heads + 2 * kv, hd)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if c["norm"]:
        q, k = _normed(q, s["qw"].double()), _normed(k, s["kw"].double())
    cs = s["rope"].double()[at][:, None]
    q, k = _turned(q, cs).float(), _turned(k, cs)
    # the blocks that the rows reach, [segment][block][16 positions]
    first, nb = pos // BLOCK, (c["rows"] + BLOCK - 2) // BLOCK + 1
    block = first[:, None] + torch.arange(nb, device="cuda")
    p = block[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    new, old = (p >= pos[:, None, None]) & (p < (pos + rows)[:, None, None]), p < pos[:, None, None]
    used = new.any(-1)
    src = (row[:, None, None] + p - pos[:, None, None]).clamp(0, s["total"] - 1)
    page = table[slot[:, None], (block // 4).clamp(max=table.shape[1] - 1)].clamp(min=0)
    page, sub = page[used], (block % 4)[used]
    new, old, src = new[used], old[used], src[used]
    out = {"q": q.reshape(s["total"], -1)}
    for which, x in (("k", k), ("v", v)):
        codes = s[which + "_codes"]
        if which == "k":
            codes = codes.view(len(codes), kv, 4, BLOCK, hd)
        had = (codes[page, :, sub] if which == "k" else codes[page, :, sub].transpose(2, 3)).double() - 128
        had_scale = s[which + "_scale"][page, :, sub].double()[..., None, None]
        x = x[src].transpose(1, 2)                                              # [blocks, kv, 16, hd]
        n, o = new[:, None, :, None], old[:, None, :, None]
        top = torch.where(n, x.abs(), 0.0).amax((2, 3), keepdim=True)
        m, e = torch.frexp(top / 127)
        scale = torch.exp2(torch.where(m == 0.5, e - 1, e).clamp(min=LOW).double())
        scale = torch.where(o.any(2, keepdim=True), torch.maximum(scale, had_scale), scale)
        now = torch.where(n, torch.round(x / scale), torch.where(o, torch.round(had * had_scale / scale), had))
        b = (now + 128).to(torch.uint8)
        codes[page, :, sub] = b if which == "k" else b.transpose(2, 3)
        s[which + "_scale"][page, :, sub] = scale[..., 0, 0].float()
        value = (now * scale).float().transpose(1, 2)                           # [blocks, 16, kv, hd]
        out[which] = value[new | old].reshape(-1, kv * hd)
    return out


def _run_attend(s):
    heads, kv, hd = s["shape"]
    c, segs = s["case"], s["segs"].long()
    slot, pos, row, rows = segs.unbind(1)
    n, grp, most = len(segs), heads // kv, c["rows"]
    t = (c["count"] + PAGE - 1) // PAGE
    page = s["table"].long()[slot, :t].clamp(min=0)
    k = (s["k_codes"].float()[page] - 128).view(n, t, kv, 4, BLOCK, hd) * s["k_scale"][page][..., None, None]
    k = k.permute(0, 2, 1, 3, 4, 5).reshape(n, kv, t * PAGE, hd)
    v = (s["v_codes"].float()[page] - 128) * s["v_scale"][page][..., None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(n, kv, t * PAGE, hd)
    # the segments' rows, padded to the longest
    i = torch.arange(most, device="cuda")
    live = i < rows[:, None]
    src = (row[:, None] + i).clamp(max=s["total"] - 1)
    q = s["q"][src].view(n, most, kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, most * grp, hd)
    x = torch.matmul(q * (1 / math.sqrt(hd)), k.transpose(2, 3).contiguous()).view(n, kv, most, grp, t * PAGE)
    at, p = torch.arange(t * PAGE, device="cuda"), (pos[:, None] + i)[..., None]
    seen = at <= p
    if c["window"]:
        seen = seen & (at > p - c["window"])
    x = x.masked_fill_(~seen[:, None, :, None], -math.inf)
    x = torch.exp(x.sub_(x.amax(-1, keepdim=True)))
    y = torch.matmul((x / x.sum(-1, keepdim=True)).view(n, kv, most * grp, t * PAGE), v)
    y = y.view(n, kv, most, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, most, heads * hd)
    return y[live]


def run(state):
    if own:
        return _run_own(state)
    return _run_append(state) if state["case"]["kind"] == "append" else _run_attend(state)


# ------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    heads, kv, hd = SHAPES[case["shape"]]
    return _exact_append(s, case, heads, kv, hd) if case["kind"] == "append" else _exact_attend(s, case, heads, kv, hd)


def _cached(s, slot, count):
    """K and V of a slot's first `count` positions, each [count, kv, hd], and the pages that hold them."""
    pages = s["table"][slot, :(count + PAGE - 1) // PAGE].long()
    k = s["k_codes"][pages].double() - 128
    v = (s["v_codes"][pages].double() - 128).permute(0, 1, 2, 4, 3)
    ks, vs = (s[n][pages].double().repeat_interleave(BLOCK, 2).unsqueeze(-1) for n in ("k_scale", "v_scale"))
    k, v = k * ks, v.reshape(k.shape) * vs
    return tuple(x.transpose(1, 2).reshape(-1, k.shape[1], k.shape[3])[:count] for x in (k, v))


def _exact_attend(s, case, heads, kv, hd):
    out = torch.empty(s["total"], heads, hd, dtype=torch.float64, device="cuda")
    for slot, pos, row, rows in s["segs"].tolist():
        k, v = _cached(s, slot, pos + rows)
        last = torch.arange(pos, pos + rows, device="cuda")[:, None]
        at = torch.arange(pos + rows, device="cuda")[None]
        hidden = (at > last) | ((last - at >= case["window"]) if case["window"] else False)
        q = s["q"][row:row + rows].double().view(rows, heads, hd)
        for h in range(heads):
            x = q[:, h] @ k[:, h * kv // heads].t().contiguous() / hd ** 0.5
            out[row:row + rows, h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ v[:, h * kv // heads].contiguous()
    return out.reshape(s["total"], -1)


def _exact_append(s, case, heads, kv, hd):
    parts = s["qkv"].double().view(s["total"], -1, hd).split((heads, kv, kv), 1)
    q, k, v = parts
    if case["norm"]:
        q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) / hd + EPS) * s["qw"].double()
        k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) / hd + EPS) * s["kw"].double()
    out = {"q": [], "k": [], "v": []}
    for slot, pos, row, rows in s["segs"].tolist():
        turn = torch.view_as_complex(s["rope"][pos:pos + rows].double())[:, None]

        def rotated(x):
            z = torch.complex(x[row:row + rows, :, :hd // 2], x[row:row + rows, :, hd // 2:]) * turn
            return torch.cat((z.real, z.imag), -1)

        out["q"].append(rotated(q).reshape(rows, -1))
        first = pos // BLOCK * BLOCK
        old = _cached(s, slot, pos)
        pages = s["table"][slot].long()
        for name, was, now in (("k", old[0], rotated(k)), ("v", old[1], v[row:row + rows])):
            x = torch.cat((was[first:], now))                     # from the first block's start on
            pad = -len(x) % BLOCK
            x = torch.cat((x, x.new_zeros(pad, kv, hd))).view(-1, BLOCK, kv, hd)
            fresh = x.clone()
            fresh[0, :pos - first] = 0
            step = torch.full((len(x), kv), 2.0 ** LOW, dtype=torch.float64, device="cuda")
            for _ in range(HIGH - LOW):                           # the least power of two that holds the new values
                step = torch.where(fresh.abs().amax((1, 3)) > 127 * step, 2 * step, step)
            if pos > first:
                step[0] = torch.maximum(step[0], s[name + "_scale"][pages[first // PAGE], :, first % PAGE // BLOCK].double())
            step = step[:, None, :, None]
            x = (torch.round(x / step) * step).reshape(-1, kv * hd)
            out[name].append(x[:len(x) - pad])
    return {n: torch.cat(v) for n, v in out.items()}


# ------------------------------------------------------------------ the rest

def work(case):
    heads, kv, hd = SHAPES[case["shape"]]
    bytes_ = flops = 0
    for before, rows in _lengths(case):
        if case["kind"] == "append":
            back = before % BLOCK
            bytes_ += rows * hd * (8 * heads + 8 * kv + 2 * kv) + back * 2 * kv * hd + (back + rows) * 8 * kv * hd
            flops += 3 * rows * hd * (heads + kv)
        else:
            w = case["window"] or 1 << 40
            seen = sum(min(w, before + i + 1) for i in range(rows))
            bytes_ += 2 * kv * hd * min(before + rows, w + rows - 1) + 8 * rows * heads * hd
            flops += 4 * heads * hd * seen
    return {"bytes": bytes_, "flops": flops}
