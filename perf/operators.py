"""The operators of a layer between its q/k/v projections and its output
projection over an 8-bit K/V cache, as cases to be timed: the rotation of q and
k by positions of three axes, the cache's append and read, attention over it
(with the weight that every slot receives), and the eviction of slots by that
weight.  Head shapes are those of oi.synth.CONFIGS.

The cache holds one signed byte per value and one exponent per (kv head, block
of slots), apart for K and V: value = code * 2^exponent, code in [-127, 127],
exponent in [-24, 10].  In memory, one buffer: K codes [kv_head][slot][dim],
V codes [kv_head][slot / 64][dim][slot % 64], K exponents, V exponents
[kv_head][slot / block].

A case runs in its plain form (elementary torch operations) or, where `own` is
set, through the framework's calls.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EMIN, EMAX = -24, 10
DTYPES = {"f32": torch.float32, "f16": torch.float16}
CODES = {"f32": 0, "f16": 1}  # the type ids of include/oi.h


def listed():
    return [
        # one token of a dense 8B-class layer: a few microseconds, where the launch counts
        dict(name="rope-token", op="rope", heads=32, kv_heads=8, head_dim=128, rotary=128, time=24, height=20, width=20,
             interleaved=True, gate=False, n=1, type="f32", out="f32"),
        # a prompt with images read by a gated full-attention layer, q beside its gate, f16 for the matrix cores
        dict(name="rope-prompt", op="rope", heads=16, kv_heads=2, head_dim=256, rotary=64, time=11, height=11, width=10,
             interleaved=True, gate=True, n=2311, type="f32", out="f16"),
        # one decoded token's K and V into a partly filled block
        dict(name="append-token", op="append", kv_heads=8, head_dim=128, block=32, n=1, past=4099, type="f32"),
        # a long document's K and V behind a short preamble, no round slots
        dict(name="append-prompt", op="append", kv_heads=8, head_dim=128, block=64, n=8001, past=37, type="f16"),
        # the last few slots of a gated layer's cache, for a check or a rollback
        dict(name="read-tail", op="read", kv_heads=2, head_dim=256, block=16, slot=4075, n=21, type="f32"),
        # a whole long conversation's cache on its way to a state file
        dict(name="read-long", op="read", kv_heads=8, head_dim=128, block=64, slot=0, n=40001, type="f32"),
        # a decode step of a dense 8B-class layer early in a conversation
        dict(name="attn-token", op="attn", heads=32, kv_heads=8, head_dim=128, block=32, n=1, past=1030, type="f32",
             mass=False),
        # a decode step deep in a long context, with the weights that an eviction goes by
        dict(name="attn-token-long", op="attn", heads=32, kv_heads=4, head_dim=128, block=64, n=1, past=100003,
             type="f32", mass=True),
        # a draft of six tokens verified by a gated full-attention layer
        dict(name="attn-verify", op="attn", heads=16, kv_heads=2, head_dim=256, block=64, n=6, past=8190, type="f32",
             mass=False),
        # a prompt chunk of a dense 8B-class layer behind 6000 positions, weights accumulated
        dict(name="attn-prompt", op="attn", heads=32, kv_heads=8, head_dim=128, block=64, n=2047, past=6001,
             type="f16", mass=True),
        # a sliding conversation cut to half its slots
        dict(name="evict-half", op="evict", kv_heads=2, head_dim=256, block=32, n=4096, keep=2045, first=4, last=256),
        # a long document cut to what a session keeps
        dict(name="evict-long", op="evict", kv_heads=8, head_dim=128, block=64, n=40960, keep=8192, first=16,
             last=1024),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attn", "attn", "attn", "evict"])
    hd = rng.choice([128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    block = rng.choice([16, 32, 64])
    if op == "rope":
        rot = rng.choice([64, 128, hd])
        third = rot // 6
        return dict(op=op, heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv, head_dim=hd, rotary=rot, time=rot // 2 - 2 * third,
                    height=third, width=third,
                    interleaved=rng.random() < 0.5, gate=rng.random() < 0.5, n=_log_int(rng, 1, 8192),
                    type=rng.choice(["f32", "f16"]), out=rng.choice(["f32", "f16"]))
    if op == "append":
        return dict(op=op, kv_heads=kv, head_dim=hd, block=block, n=_log_int(rng, 1, 16000),
                    past=rng.choice([0, _log_int(rng, 1, 20000)]), type=rng.choice(["f32", "f16"]))
    if op == "read":
        return dict(op=op, kv_heads=kv, head_dim=hd, block=block, slot=rng.choice([0, _log_int(rng, 1, 5000)]),
                    n=_log_int(rng, 1, 30000), type=rng.choice(["f32", "f16"]))
    if op == "evict":
        n = _log_int(rng, 300, 60000)
        keep = rng.randint(n // 8, n - 1)
        first = rng.randint(0, 32)
        return dict(op=op, kv_heads=kv, head_dim=hd, block=block, n=n, keep=keep, first=first,
                    last=rng.randint(0, (keep - first) // 2))
    g = rng.choice([1, 2, 4, 8])
    t = rng.choice(["f32", "f16"])
    n = rng.choice([1, _log_int(rng, 2, 16), _log_int(rng, 17, 1500)])
    past = rng.choice([0, _log_int(rng, 1, 4000), _log_int(rng, 4001, 100000 if n <= 16 else 8000)])
    if n > 16:  # no more work than the largest listed case
        while g > 1 and kv * g * hd * n * (past + n) > 3e10:
            g //= 2
        n = max(17, min(n, int(3e10 / (kv * g * hd * (past + n)))))
    return dict(op=op, heads=kv * g, kv_heads=kv, head_dim=hd, block=block, n=n, past=past, type=t,
                mass=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --

def _gen(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + what * 7919 + 12345) & 0x7FFFFFFFFFFF)
    return g


def _normal(seed, what, *shape, dtype="f32", scale=1.0):
    x = torch.randn(*shape, generator=_gen(seed, what), device=DEV)
    return (x if scale == 1.0 else x * scale).to(DTYPES[dtype])


def _rows(seed, what, *shape, dtype="f32"):
    """K or V rows [..., head_dim]: N(0, 1), each token with a size of its own,
    and a few dimensions several times larger, as K's are in trained models."""
    x = torch.randn(*shape, generator=_gen(seed, what), device=DEV)
    size = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=_gen(seed, what + 100), device=DEV))
    wide = 1 + 5 * (torch.rand(shape[-1], generator=_gen(seed, what + 200), device=DEV) < 0.03).float()
    return (x * size * wide).to(DTYPES[dtype])


class _Cache:
    """One buffer in the layout above, and its parts."""

    def __init__(self, case, capacity):
        h, d, b = case["kv_heads"], case["head_dim"], case["block"]
        self.h, self.d, self.b, self.cap = h, d, b, capacity
        n, m = h * capacity * d, h * capacity // b
        self.buf = torch.zeros((2 * n + 2 * m + 255) // 256 * 256, dtype=torch.uint8, device=DEV)
        i8 = self.buf.view(torch.int8)
        self.kc = i8[:n].view(h, capacity, d)
        self.vc = i8[n:2 * n].view(h, capacity // 64, d, 64)
        self.ke = i8[2 * n:2 * n + m].view(h, capacity // b)
        self.ve = i8[2 * n + m:2 * n + 2 * m].view(h, capacity // b)


def _capacity(n):
    return (n + 63) // 64 * 64


def _fill(case, seed, n, capacity):
    """A cache of n slots of random K and V as an append of all n leaves it."""
    c = _Cache(case, capacity)
    if n:
        for what, codes, exps in ((1, c.kc, c.ke), (2, c.vc, c.ve)):
            x = torch.zeros(c.h, capacity, c.d, device=DEV)
            x[:, :n] = _rows(seed, what, c.h, n, c.d)
            xb = x.view(c.h, capacity // c.b, c.b * c.d)
            m, k = torch.frexp(xb.abs().amax(-1))
            e = torch.where(m == 0, torch.full_like(k, EMIN), k - 7 + (m > 127 / 128).int()).clamp(EMIN, EMAX)
            q = torch.round(torch.ldexp(xb, -e[..., None])).to(torch.int8).view(c.h, capacity, c.d)
            exps.copy_(e)
            codes.copy_(q if what == 1 else q.view(c.h, capacity // 64, 64, c.d).transpose(2, 3))
            del x, xb, q
    return c


def _positions(case, seed):
    """Three axes: text (the same number on each) with images of a grid inside it."""
    n = case["n"]
    t = torch.arange(n, device=DEV)
    start = int(torch.randint(0, 100000, (1,), generator=_gen(seed, 21), device=DEV))
    image = (t // 256) % 2 == 1
    p = torch.stack([torch.where(image, t // 256 * 256, t), torch.where(image, t // 256 * 256 + t % 256 // 16, t),
                     torch.where(image, t // 256 * 256 + t % 16, t)])
    return (p + start).to(torch.int32).contiguous()


def _sections(case):
    return [case["time"], case["height"], case["width"]]


def _rope_inputs(case, seed):
    n, h, hk, d = case["n"], case["heads"], case["kv_heads"], case["head_dim"]
    half = case["rotary"] // 2
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    return dict(q=_normal(seed, 1, n, h, (2 if case["gate"] else 1) * d, dtype=case["type"]),
                k=_normal(seed, 2, n, hk, d, dtype=case["type"]), q_norm=1 + _normal(seed, 3, d, scale=0.1),
                k_norm=1 + _normal(seed, 4, d, scale=0.1), pos=_positions(case, seed),
                inv_freq=(1e6 ** (-i / half)).float())


def _mass(case, seed, capacity):
    """What slots have received so far: most of them little, a few a lot."""
    return torch.exp(2 * torch.randn(case["kv_heads"], capacity, generator=_gen(seed, 31), device=DEV))


def prepare(case, seed):
    op = case["op"]
    s = dict(op=op, case=case)
    hk, d = case["kv_heads"], case["head_dim"]
    if op == "rope":
        s.update(_rope_inputs(case, seed))
        o = DTYPES[case["out"]]
        s.update(q_out=torch.empty(case["n"], case["heads"], d, dtype=o, device=DEV),
                 k_out=torch.empty(case["n"], hk, d, dtype=o, device=DEV))
    elif op == "append":
        n, past = case["n"], case["past"]
        b = case["block"]
        s["c"] = _fill(case, seed, past, _capacity(past + n))
        s["k"] = _rows(seed, 11, n, hk, d, dtype=case["type"])
        s["v"] = _rows(seed, 12, n, hk, d, dtype=case["type"])
        s["ko"], s["vo"] = (torch.empty(hk, past % b + n, d, device=DEV) for _ in range(2))
    elif op == "read":
        s["c"] = _fill(case, seed, case["slot"] + case["n"], _capacity(case["slot"] + case["n"]))
        s["ko"], s["vo"] = (torch.empty(hk, case["n"], d, dtype=DTYPES[case["type"]], device=DEV) for _ in range(2))
    elif op == "attn":
        n, cap = case["n"], _capacity(case["past"] + case["n"])
        s["c"] = _fill(case, seed, case["past"] + n, cap)
        s["q"] = _normal(seed, 11, n, case["heads"], d, dtype=case["type"], scale=1.5)
        s["out"] = torch.empty_like(s["q"])
        # a window of observation that has just begun: this call's weights count beside what is there
        s["mass"] = 1e-5 * _mass(case, seed, cap) if case["mass"] else None
    else:
        n, cap = case["n"], _capacity(case["n"])
        s["c"] = _fill(case, seed, n, cap)
        s["mass"] = _mass(case, seed, cap)
        s["pos"] = (torch.arange(cap, device=DEV, dtype=torch.int32) * 2 + 5).expand(hk, cap).contiguous()
        keep, kcap = case["keep"], _capacity(case["keep"])
        s["dst"] = _Cache(case, kcap)
        s["kept"] = torch.empty(hk, keep, dtype=torch.int32, device=DEV)
        s["dst_mass"] = torch.zeros(hk, kcap, device=DEV)
        s["dst_pos"] = torch.zeros(hk, kcap, dtype=torch.int32, device=DEV)
        s["ko"], s["vo"] = (torch.empty(hk, keep, d, device=DEV) for _ in range(2))
    return s


# ------------------------------------------------------------- plain forms --

def _axes(case):
    """The axis of each rotary pair: in turn while an axis' section lasts, or section after section."""
    half, s = case["rotary"] // 2, _sections(case)
    i = torch.arange(half, device=DEV)
    if case["interleaved"]:
        size = torch.tensor(s, device=DEV)
        return torch.where(i < 3 * size[i % 3], i % 3, 0)
    return (i >= s[0]).long() + (i >= s[0] + s[1]).long()


def _plain_rope(s):
    case = s["case"]
    d, half = case["head_dim"], case["rotary"] // 2
    ang = s["pos"].double().t()[:, _axes(case)] * s["inv_freq"].double()
    c, sn = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def one(x, w):
        x = x[..., :d].float()
        x = w * (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6))
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * sn, a * sn + b * c, x[..., 2 * half:]], -1).to(DTYPES[case["out"]])

    return one(s["q"], s["q_norm"]), one(s["k"], s["k_norm"])


def _codes(c, which):
    """Codes as [kv_head][slot][dim]."""
    return c.kc if which == "k" else c.vc.transpose(2, 3).reshape(c.h, c.cap, c.d)


def _values(c, which, a, b):
    """What slots a..b-1 stand for, f32 [kv_head][slot][dim]."""
    e = (c.ke if which == "k" else c.ve).repeat_interleave(c.b, 1)[:, a:b, None]
    return _codes(c, which)[:, a:b].float() * torch.exp2(e.float())


def _exponent(amax):
    """The least e with amax <= 127 * 2^e."""
    m, k = torch.frexp(amax)
    return torch.where(m == 0, torch.full_like(k, EMIN), k - 7 + (m > 127 / 128).int()).clamp(EMIN, EMAX)


def _put(c, which, slot0, codes, e):
    """Codes [kv_head][n][dim] of whole blocks from slot0, and their exponents, into the cache."""
    n = codes.shape[1]
    (c.ke if which == "k" else c.ve)[:, slot0 // c.b:(slot0 + n) // c.b] = e.to(torch.int8)
    if which == "k":
        c.kc[:, slot0:slot0 + n] = codes.to(torch.int8)
    else:
        slots = torch.arange(slot0, slot0 + n, device=DEV)
        c.vc[:, slots // 64, :, slots % 64] = codes.to(torch.int8).transpose(0, 1)


def _plain_append(s, which):
    c, n, past = s["c"], s["case"]["n"], s["case"]["past"]
    a, b = past // c.b * c.b, (past + n + c.b - 1) // c.b * c.b
    old = past - a
    x = torch.zeros(c.h, b - a, c.d, device=DEV)
    x[:, old:old + n] = s[which].float().transpose(0, 1)
    xb = x.view(c.h, -1, c.b, c.d)
    e = _exponent(xb.abs().amax((2, 3)))
    if old:
        e0 = (c.ke if which == "k" else c.ve)[:, a // c.b].int()
        e[:, 0] = torch.maximum(e[:, 0], e0)
        before = _codes(c, which)[:, a:past].float() * torch.exp2((e0 - e[:, 0]).float())[:, None, None]
    q = torch.round(xb * torch.exp2(-e.float())[..., None, None]).clamp(-127, 127).view(c.h, b - a, c.d)
    if old:
        q[:, :old] = torch.round(before)
    _put(c, which, a, q, e)
    return (q * torch.exp2(e.float()).repeat_interleave(c.b, 1)[..., None])[:, :old + n]


def _plain_attn(s):
    case, c = s["case"], s["c"]
    n, past, h, d = case["n"], case["past"], case["heads"], case["head_dim"]
    g, end = h // c.h, past + n
    k, v = _values(c, "k", 0, end), _values(c, "v", 0, end)
    q = s["q"].float().view(n, c.h, g, d).permute(1, 2, 0, 3).reshape(c.h, g * n, d)
    p = torch.bmm(q, k.transpose(1, 2)).mul_(1 / math.sqrt(d)).view(c.h, g, n, end)
    if n > 1:
        seen = torch.arange(end, device=DEV) <= past + torch.arange(n, device=DEV)[:, None]
        p.masked_fill_(~seen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = torch.bmm(p.view(c.h, g * n, end), v).view(c.h, g, n, d).permute(2, 0, 1, 3).reshape(n, h, d)
    out = o.to(s["q"].dtype)
    if not case["mass"]:
        return out
    w = p.sum((1, 2))
    s["mass"][:, :past] += w[:, :past]
    s["mass"][:, past:end] = w[:, past:]
    return out, s["mass"][:, :end]


def _plain_evict(s):
    case, c, t = s["case"], s["c"], s["dst"]
    n, keep, first, last = case["n"], case["keep"], case["first"], case["last"]
    order = torch.sort(s["mass"][:, first:n - last], dim=1, descending=True, stable=True)[1]
    middle = order[:, :keep - first - last] + first
    ends = torch.cat([torch.arange(first, device=DEV), torch.arange(n - last, n, device=DEV)])
    kept = torch.sort(torch.cat([middle, ends.expand(c.h, -1)], 1), dim=1)[0]
    heads = torch.arange(c.h, device=DEV)[:, None]
    out = []
    for which in "kv":
        x = torch.zeros(c.h, t.cap, c.d, device=DEV)
        x[:, :keep] = _values(c, which, 0, n)[heads, kept]
        e = _exponent(x.view(c.h, -1, c.b, c.d).abs().amax((2, 3)))
        scale = torch.exp2(e.float()).repeat_interleave(c.b, 1)[..., None]
        q = torch.round(x / scale)
        _put(t, which, 0, q, e)
        out.append((q * scale)[:, :keep])
    s["kept"].copy_(kept)
    s["dst_mass"][:, :keep] = s["mass"][heads, kept]
    s["dst_pos"][:, :keep] = s["pos"][heads, kept]
    return s["kept"], s["dst_mass"][:, :keep], s["dst_pos"][:, :keep], out[0], out[1]


# -------------------------------------------------------------------- calls --

def _plan(s):
    """The call's plans and workspace, made on a state's first pass and kept, as a user's program keeps them."""
    path = os.path.join(os.getcwd(), "odin-infer_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from oi import kv8, rope
    case, op = s["case"], s["op"]
    if op == "rope":
        s["plan"] = rope.RopeAxes(case["heads"], case["kv_heads"], case["head_dim"], case["rotary"], _sections(case),
                                  case["interleaved"], 1e-6)
        return
    c = s["c"]
    s["plan"] = kv8.KV8(c.h, c.d, c.cap, c.b)
    if op == "attn":
        need = s["plan"].attn_workspace_bytes(case["heads"], case["n"])
        s["ws"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    if op == "evict":
        s["dst_plan"] = kv8.KV8(c.h, c.d, s["dst"].cap, c.b)


def _own(s):
    if "plan" not in s:
        _plan(s)
    case, op = s["case"], s["op"]
    st = torch.cuda.current_stream().cuda_stream
    if op == "rope":
        d = case["head_dim"]
        qh = 2 * d if case["gate"] else d
        s["plan"].launch(case["n"], s["pos"].data_ptr(), s["inv_freq"].data_ptr(), s["q_norm"].data_ptr(),
                         s["k_norm"].data_ptr(), CODES[case["type"]], s["q"].data_ptr(), s["k"].data_ptr(),
                         CODES[case["out"]], s["q_out"].data_ptr(), s["k_out"].data_ptr(), q_head_stride=qh, stream=st)
        return s["q_out"], s["k_out"]
    plan, buf = s["plan"], s["c"].buf.data_ptr()
    if op == "append":
        # then the values that the touched blocks hold now, as the cache gives them back
        n, past, t = case["n"], case["past"], CODES[case["type"]]
        plan.append(buf, t, s["k"].data_ptr(), s["v"].data_ptr(), n, past, stream=st)
        a = past // s["c"].b * s["c"].b
        plan.read(buf, a, past + n - a, 0, s["ko"].data_ptr(), s["vo"].data_ptr(), stream=st)
        return s["ko"], s["vo"]
    if op == "read":
        plan.read(buf, case["slot"], case["n"], CODES[case["type"]], s["ko"].data_ptr(), s["vo"].data_ptr(), stream=st)
        return s["ko"], s["vo"]
    if op == "attn":
        mass = s["mass"]
        plan.attn(buf, case["heads"], CODES[case["type"]], s["q"].data_ptr(), case["n"], case["past"],
                  s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(),
                  mass=mass.data_ptr() if mass is not None else None, stream=st)
        return s["out"] if mass is None else (s["out"], mass[:, :case["past"] + case["n"]])
    keep = case["keep"]
    plan.evict(buf, s["mass"].data_ptr(), s["pos"].data_ptr(), case["n"], keep, case["first"], case["last"],
               s["dst_plan"], s["dst"].buf.data_ptr(), s["dst_mass"].data_ptr(), s["dst_pos"].data_ptr(),
               s["kept"].data_ptr(), stream=st)
    s["dst_plan"].read(s["dst"].buf.data_ptr(), 0, keep, 0, s["ko"].data_ptr(), s["vo"].data_ptr(), stream=st)
    return s["kept"], s["dst_mass"][:, :keep], s["dst_pos"][:, :keep], s["ko"], s["vo"]


def run(s):
    if own:
        return _own(s)
    op = s["op"]
    if op == "rope":
        return _plain_rope(s)
    if op == "append":
        return _plain_append(s, "k"), _plain_append(s, "v")
    if op == "read":
        c, a, b = s["c"], s["case"]["slot"], s["case"]["slot"] + s["case"]["n"]
        t = DTYPES[s["case"]["type"]]
        return _values(c, "k", a, b).to(t), _values(c, "v", a, b).to(t)
    return _plain_attn(s) if op == "attn" else _plain_evict(s)


# --------------------------------------------------------------------- work --

SIZE = {"f32": 4, "f16": 2}


def work(case):
    op, hk, d = case["op"], case["kv_heads"], case["head_dim"]
    n = case["n"]
    if op == "rope":
        e = n * (case["heads"] + hk) * d
        return {"bytes": e * (SIZE[case["type"]] + SIZE[case["out"]]) + 12 * n + 2 * case["rotary"] + 8 * d,
                "flops": 10 * e}
    if op == "append":  # in, codes out, and the values read back
        back = case["past"] % case["block"] + n
        return {"bytes": 2 * hk * d * (n * (SIZE[case["type"]] + 1) + back * 5), "flops": 6 * hk * d * n}
    if op == "read":
        return {"bytes": 2 * hk * d * n * (1 + SIZE[case["type"]]), "flops": 2 * hk * d * n}
    if op == "attn":
        h, end = case["heads"], case["past"] + n
        seen = n * case["past"] + n * (n + 1) // 2
        return {"bytes": 2 * hk * end * d + 2 * n * h * d * SIZE[case["type"]] + (8 * hk * end if case["mass"] else 0),
                "flops": 4 * h * d * seen}
    keep = case["keep"]  # masses in; kept slots, masses, positions and codes; the values read back
    return {"bytes": hk * (4 * n + keep * (4 + 8 + 8)) + 2 * hk * d * keep * (1 + 1 + 5), "flops": 4 * hk * d * keep}


# ------------------------------------------------------- in 64 bits, apart --

def _step(amax):
    """2^e for the least e in [EMIN, EMAX] with amax <= 127 * 2^e, counted off a list of all of them."""
    bounds = 127.0 * torch.exp2(torch.arange(EMIN, EMAX, device=DEV, dtype=torch.float64))
    return torch.exp2((EMIN + (amax[..., None] > bounds).sum(-1)).double())


def _kept_values(c, which, head, n):
    """Slots 0..n-1 of one head in 64 bits, [slot][dim]."""
    if which == "k":
        codes, e = c.kc[head, :n], c.ke[head]
    else:
        codes, e = c.vc[head].permute(0, 2, 1).flatten(0, 1)[:n], c.ve[head]
    return codes.double() * torch.exp2(e.double())[torch.arange(n, device=DEV) // c.b, None]


def _regroup(x, b, old_step=None):
    """Rows [slot][dim] in blocks of b (the first of them at least with old_step), rounded to their blocks' steps."""
    n = x.shape[0]
    which = torch.arange(n, device=DEV) // b
    top = torch.zeros(int(which[-1]) + 1, dtype=torch.float64, device=DEV)
    top = top.scatter_reduce(0, which, x.abs().amax(1), "amax")
    step = _step(top)
    if old_step is not None:
        step[0] = max(step[0], old_step)
    step = step[which, None]
    return (x / step).round().clamp(-127, 127) * step


def exact(case, seed):
    op, hk, d = case["op"], case["kv_heads"], case["head_dim"]
    if op == "rope":
        i, half, sec = _rope_inputs(case, seed), case["rotary"] // 2, _sections(case)
        axis = [0] * half
        for p in range(half):
            if case["interleaved"]:
                axis[p] = p % 3 if p < 3 * sec[p % 3] else 0
            else:
                axis[p] = 0 if p < sec[0] else 1 if p < sec[0] + sec[1] else 2
        z = torch.polar(torch.ones(case["n"], half, dtype=torch.float64, device=DEV),
                        torch.stack([i["pos"][a].double() for a in axis], 1) * i["inv_freq"].double())

        def turned(x, w):
            x = x[..., :d].double()
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + 1e-6) * w.double()
            y = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z[:, None]
            return torch.cat([y.real, y.imag, x[..., 2 * half:]], -1)

        return turned(i["q"], i["q_norm"]), turned(i["k"], i["k_norm"])
    s = prepare(case, seed)
    c, n = s["c"], case["n"]
    if op == "append":
        past, out = case["past"], []
        a = past // c.b * c.b
        for which in "kv":
            heads = []
            for h in range(hk):
                x = torch.cat([_kept_values(c, which, h, past)[a:], s[which][:, h].double()])
                e = (c.ke if which == "k" else c.ve)[h, a // c.b].double()
                heads.append(_regroup(x, c.b, torch.exp2(e) if past > a else None))
            out.append(torch.stack(heads))
        return tuple(out)
    if op == "read":
        a = case["slot"]
        return tuple(torch.stack([_kept_values(c, w, h, a + n)[a:] for h in range(hk)]) for w in "kv")
    if op == "attn":
        past, g = case["past"], case["heads"] // hk
        end = past + n
        limit = past + torch.arange(n, device=DEV)
        out = torch.empty(n, case["heads"], d, dtype=torch.float64, device=DEV)
        mass = None
        if case["mass"]:
            mass = s["mass"][:, :end].double()
            mass[:, past:] = 0
        for h in range(hk):
            k, v = _kept_values(c, "k", h, end), _kept_values(c, "v", h, end)
            for r in range(h * g, (h + 1) * g):
                x = s["q"][:, r].double() @ k.t() / math.sqrt(d)
                x[torch.arange(end, device=DEV)[None] > limit[:, None]] = -math.inf
                p = torch.softmax(x, 1)
                out[:, r] = p @ v
                if mass is not None:
                    mass[h] += p.sum(0)
        return out if mass is None else (out, mass)
    keep, first, last = case["keep"], case["first"], case["last"]
    kept, ko, vo = [], [], []
    for h in range(hk):
        m = s["mass"][h, :n].double()
        m[:first] = math.inf
        m[n - last:] = math.inf
        slots = torch.argsort(-m, stable=True)[:keep].sort()[0]
        kept.append(slots)
        ko.append(_regroup(_kept_values(c, "k", h, n)[slots], c.b))
        vo.append(_regroup(_kept_values(c, "v", h, n)[slots], c.b))
    kept = torch.stack(kept)
    return (kept.int(), s["mass"].gather(1, kept).double(), s["pos"].gather(1, kept), torch.stack(ko), torch.stack(vo))
