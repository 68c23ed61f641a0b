"""What a server of many requests needs between a layer's projections, as cases
to be timed: the pages of a pool given to requests and the slot of every packed
row, the append of packed K and V to a paged cache, attention of the newest
tokens of many requests, and attention of packed prompts.  Head shapes are those
of oi.synth.CONFIGS.

The cache is a pool of pages of `page` slots, binary16, one buffer: K
[n_pages][kv_head][page][dim], then V [n_pages][kv_head][page / 8][dim][8].  A
request's slot j lies in page table[request][j / page] at j % page.

A case runs in its plain form (elementary torch operations) or, where `own` is
set, through the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16}
CODES = {"f32": 0, "f16": 1}  # the type ids of include/oi.h
SIZE = {"f32": 4, "f16": 2}
TOP = 65504.0


# Lengths of a case's requests: `mix` is the seed of the draw, so that a case stands for one set of them.
# plan: past in past_lo .. past_hi, new in new_lo .. new_hi.  tokens: lengths in lo .. hi (the first is hi).
# prompts: new tokens in lo .. hi (the first is hi) behind past_lo .. past_hi.

def listed():
    return [
        # one step of a busy server: a token for each of 61 requests; the pages are taken and, as after a
        # rejected draft, given back
        dict(name="plan-step", op="plan", seqs=61, page=16, past_lo=1, past_hi=4000, new_lo=1, new_hi=1, pad=3, mix=1),
        # a burst of requests whose prompts are read in one batch, and a pool that does not hold the last of them
        dict(name="plan-prompts", op="plan", seqs=300, page=64, past_lo=0, past_hi=700, new_lo=1, new_hi=180, pad=64,
             mix=2),
        # the K and V of one decoded token of each of 64 requests
        dict(name="append-step", op="append", kv_heads=8, head_dim=128, page=16, seqs=64, lo=1, hi=1, past_hi=4000,
             pad=0, type="f32", mix=3),
        # the K and V of packed prompts, with rows of padding behind them
        dict(name="append-prompts", op="append", kv_heads=8, head_dim=128, page=64, seqs=11, lo=90, hi=2501,
             past_hi=500, pad=61, type="f16", mix=4),
        # a decode step of one conversation, early: a few microseconds, where the launch counts
        dict(name="tokens-one", op="tokens", heads=32, kv_heads=8, head_dim=128, page=16, seqs=1, n=1, lo=1031, hi=1031,
             type="f32", mix=5),
        # a decode step of a server's batch, lengths from a greeting to a long conversation
        dict(name="tokens-batch", op="tokens", heads=32, kv_heads=8, head_dim=128, page=64, seqs=48, n=1, lo=17, hi=9001,
             type="f16", mix=6),
        # drafts of five tokens verified for 24 requests
        dict(name="tokens-draft", op="tokens", heads=32, kv_heads=4, head_dim=128, page=32, seqs=24, n=5, lo=200,
             hi=3501, type="f16", mix=7),
        # a gated full-attention layer: two long documents (120001 and 99785 slots) beside a short request (2729)
        dict(name="tokens-long", op="tokens", heads=16, kv_heads=2, head_dim=256, page=64, seqs=3, n=1, lo=900,
             hi=120001, type="f32", mix=8),
        # short questions read together
        dict(name="prompts-short", op="prompts", heads=32, kv_heads=4, head_dim=128, page=16, seqs=9, lo=5, hi=301,
             past_lo=0, past_hi=0, type="f16", mix=9),
        # the last lines of long documents whose beginnings are cached
        dict(name="prompts-tail", op="prompts", heads=32, kv_heads=8, head_dim=128, page=64, seqs=2, lo=19, hi=77,
             past_lo=30000, past_hi=50000, type="f16", mix=10),
        # chunks of three prompts in a gated full-attention layer, f32 throughout
        dict(name="prompts-chunk", op="prompts", heads=16, kv_heads=2, head_dim=256, page=32, seqs=3, lo=250, hi=700,
             past_lo=1000, past_hi=5000, type="f32", mix=11),
        # a batch of whole prompts of a dense 8B-class model
        dict(name="prompts-large", op="prompts", heads=32, kv_heads=8, head_dim=128, page=64, seqs=6, lo=900, hi=5003,
             past_lo=0, past_hi=0, type="f16", mix=12),
    ]


LIMIT = 3.5e11  # 4 * heads * dim * pairs of a row and a slot: below the largest listed case


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "append", "tokens", "tokens", "prompts", "prompts", "prompts"])
    page, mix = rng.choice([16, 32, 64]), rng.randint(100, 10 ** 6)
    if op == "plan":
        new = rng.choice([1, _log_int(rng, 2, 8), _log_int(rng, 9, 200)])
        return dict(op=op, seqs=_log_int(rng, 1, 400), page=page, past_lo=0, past_hi=_log_int(rng, 1, 5000),
                    new_lo=rng.choice([0, 1]), new_hi=new, pad=rng.choice([0, rng.randint(1, 99)]), mix=mix)
    hd, kv = rng.choice([128, 128, 256]), rng.choice([1, 2, 4, 8])
    t = rng.choice(["f32", "f16"])
    if op == "append":
        return dict(op=op, kv_heads=kv, head_dim=hd, page=page, seqs=_log_int(rng, 1, 80), lo=1,
                    hi=rng.choice([1, _log_int(rng, 2, 150)]), past_hi=_log_int(rng, 1, 3000),
                    pad=rng.choice([0, rng.randint(1, 70)]), type=t, mix=mix)
    g = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "tokens":
        return dict(op=op, heads=kv * g, kv_heads=kv, head_dim=hd, page=page, seqs=_log_int(rng, 1, 64),
                    n=rng.choice([1, 1, rng.randint(2, 8)]), lo=1, hi=_log_int(rng, 1, 12000), type=t, mix=mix)
    case = dict(op=op, heads=kv * g, kv_heads=kv, head_dim=hd, page=page, seqs=_log_int(rng, 1, 12), lo=1,
                hi=_log_int(rng, 1, 3000), past_lo=0, past_hi=rng.choice([0, _log_int(rng, 1, 8000)]), type=t, mix=mix)
    while work(case)["flops"] > LIMIT:
        case["hi"] = case["hi"] * 3 // 4
        case["past_hi"] = case["past_hi"] * 3 // 4
    return case


def _lengths(case):
    """(past, new) of every request."""
    r, n = random.Random(case["mix"]), case["seqs"]
    op = case["op"]
    if op == "plan":
        past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(n)]
        return past, [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
    new = [case["hi"]] + [_log_int(r, case["lo"], case["hi"]) for _ in range(n - 1)]
    if op == "tokens":  # lengths after the append of this step's tokens
        return [max(x, case["n"]) - case["n"] for x in new], [case["n"]] * n
    lo = case.get("past_lo", 0)
    return [r.randint(lo, case["past_hi"]) for _ in range(n)], new


def _prefix(xs):
    out = [0]
    for x in xs:
        out.append(out[-1] + x)
    return out


def _pages(slots, page):
    return (slots + page - 1) // page


# ------------------------------------------------------------------ inputs --

def _gen(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + what * 7919 + 54321) & 0x7FFFFFFFFFFF)
    return g


def _ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device=DEV)


def _rows(seed, what, *shape, dtype="f32"):
    """K or V rows [..., head_dim]: N(0, 1), each token with a size of its own,
    and a few dimensions several times larger, as K's are in trained models."""
    x = torch.randn(*shape, generator=_gen(seed, what), device=DEV)
    size = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=_gen(seed, what + 100), device=DEV))
    wide = 1 + 5 * (torch.rand(shape[-1], generator=_gen(seed, what + 200), device=DEV) < 0.03).float()
    return (x * size * wide).to(DTYPES[dtype])


class _Pool:
    """The buffer in the layout above and its parts, in random values; the pages of requests that hold
    `held` slots, in no order, some pages nobody's."""

    def __init__(self, case, seed, held):
        h, d, p = case["kv_heads"], case["head_dim"], case["page"]
        counts = [_pages(x, p) for x in held]
        first = _prefix(counts)
        self.h, self.d, self.p, self.n = h, d, p, first[-1] + 5
        self.width = max(counts) + 2
        one = self.n * h * p * d
        self.buf = torch.empty((2 * one + 127) // 128 * 128, dtype=torch.float16, device=DEV)
        self.k = self.buf[:one].view(self.n, h, p, d)
        self.v = self.buf[one:2 * one].view(self.n, h, p // 8, d, 8)
        self.k.copy_(_rows(seed, 1, self.n, h, p, d, dtype="f16"))
        self.v.copy_(_rows(seed, 2, self.n, h, p // 8, 8, d, dtype="f16").transpose(3, 4))
        order = torch.randperm(self.n, generator=_gen(seed, 3), device=DEV).int()
        self.table = torch.zeros(len(held), self.width, dtype=torch.int32, device=DEV)
        for i, c in enumerate(counts):
            self.table[i, :c] = order[first[i]:first[i] + c]


def prepare(case, seed):
    op = case["op"]
    past, new = _lengths(case)
    total = sum(new)
    s = dict(op=op, case=case)
    if op == "plan":
        # a pool in which the requests' pages lie anywhere; the last few requests of a burst may not fit
        p, n = case["page"], case["seqs"]
        held = [_pages(x, p) for x in past]
        want = sum(_pages(x + y, p) for x, y in zip(past, new)) - sum(held)
        room = want if case["new_hi"] <= 8 else want - want // 20
        room = max(room, 1 - sum(held))  # a pool has a page where nothing is held and nothing asked for
        s["n_pages"] = sum(held) + room
        order = torch.randperm(s["n_pages"], generator=_gen(seed, 3), device=DEV).int()
        s["width"] = max(_pages(x + y, p) for x, y in zip(past, new)) + 3
        s["table"] = torch.zeros(n, s["width"], dtype=torch.int32, device=DEV)
        first = _prefix(held)
        for i, c in enumerate(held):
            s["table"][i, :c] = order[first[i]:first[i] + c]
        s["free"] = torch.cat([order[first[-1]:], order[:first[-1]]]).contiguous()
        s["n_free"] = _ints([room])
        # the same lengths in another order for another seed
        perm = torch.randperm(n, generator=_gen(seed, 4), device=DEV)
        s["table"] = s["table"][perm].contiguous()
        s["past"], s["new"] = _ints(past)[perm].contiguous(), _ints(new)[perm].contiguous()
        s["n_rows"] = total + case["pad"]
        rows = max(1, s["n_rows"])
        s["lens"], s["starts"] = (torch.empty(n + i, dtype=torch.int32, device=DEV) for i in (0, 1))
        s["slots"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        s["pos"] = torch.empty(3, rows, dtype=torch.int32, device=DEV)
        return s
    end = [x + y for x, y in zip(past, new)]
    s["c"] = c = _Pool(case, seed, end)
    hk, d = case["kv_heads"], case["head_dim"]
    if op == "append":
        n = total + case["pad"]
        s["k"] = _rows(seed, 11, n, hk, d, dtype=case["type"])
        s["v"] = _rows(seed, 12, n, hk, d, dtype=case["type"])
        slots = torch.full((n,), -1, dtype=torch.int32, device=DEV)
        at = _prefix(new)
        for i, (x, y) in enumerate(zip(past, new)):
            j = torch.arange(x, x + y, device=DEV)
            slots[at[i]:at[i + 1]] = c.table[i][j // c.p] * c.p + (j % c.p).int()
        s["slots"] = slots
        return s
    s["past"], s["new"] = past, new
    s["lens"], s["starts"] = _ints(end), _ints(_prefix(new))
    s["q"] = (1.5 * torch.randn(total, case["heads"], d, generator=_gen(seed, 11), device=DEV)).to(DTYPES[case["type"]])
    s["out"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------- plain forms --

def _plain_plan(s):
    case, width, rows = s["case"], s["width"], s["n_rows"]
    p, n = case["page"], case["seqs"]
    past, new, table, free, n_free = (s[x].long() for x in ("past", "new", "table", "free", "n_free"))
    before, after = (past + p - 1) // p, (past + new + p - 1) // p
    end = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(end[:1]), end])
    fits = (end <= rows) & (past + new <= width * p)
    need = torch.where(fits, after - before, 0)
    run = torch.cumsum(need, 0)
    given = fits & ((need == 0) | (run <= n_free))
    # a granted request's new entries come off the end of the list, in the requests' order
    col = torch.arange(width, device=DEV)
    fresh = given[:, None] & (col >= before[:, None]) & (col < after[:, None])
    place = n_free - 1 - ((run - need)[:, None] + col - before[:, None])
    table = torch.where(fresh, free[place.clamp(0, s["n_pages"] - 1)], table)
    lens = torch.where(given, past + new, 0)
    t = torch.arange(rows, device=DEV)
    who = (t[:, None] >= end).sum(1)
    of = who.clamp(max=n - 1)
    j = past[of] + t - starts[of]
    live = (who < n) & given[of]
    slots = torch.where(live, table[of, (j // p).clamp(0, width - 1)] * p + j % p, -1)
    pos = torch.where(live, j, 0)
    s["table"].copy_(table)
    # given back: the list and its count are what they were
    return s["table"], lens.int(), starts.clamp(max=rows).int(), slots.int(), pos.int().expand(3, rows), s["free"], s["n_free"]


def _stored(x):
    """f32 or f16 rows as the cache holds them: to nearest even, nothing infinite, no NaN."""
    x = x.float()
    return torch.where(x == x, x.clamp(-TOP, TOP), 0.0).half()


def _plain_append(s):
    c = s["c"]
    slot = s["slots"].long()
    live = torch.nonzero(slot >= 0).squeeze(1)
    slot = slot[live]
    page, off = slot // c.p, slot % c.p
    c.k[page, :, off] = _stored(s["k"])[live]
    c.v[page, :, off // 8, :, off % 8] = _stored(s["v"])[live]
    return c.k, c.v


def _request(c, i, end):
    """K and V of request i, f32 [kv_head][slot][dim]."""
    pages = c.table[i, :_pages(end, c.p)].long()
    k = c.k[pages].transpose(0, 1).reshape(c.h, -1, c.d)[:, :end]
    v = c.v[pages].permute(1, 0, 2, 4, 3).reshape(c.h, -1, c.d)[:, :end]
    return k.float(), v.float()


def _plain_attn(s):
    case, c = s["case"], s["c"]
    h, d = case["heads"], case["head_dim"]
    g, at = h // c.h, _prefix(s["new"])
    out = torch.empty_like(s["q"])
    for i, (past, n) in enumerate(zip(s["past"], s["new"])):
        end = past + n
        k, v = _request(c, i, end)
        q = s["q"][at[i]:at[i + 1]].float().view(n, c.h, g, d).permute(1, 2, 0, 3).reshape(c.h, g * n, d)
        p = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(d)).view(c.h, g, n, end)
        if n > 1:
            seen = torch.arange(end, device=DEV) <= past + torch.arange(n, device=DEV)[:, None]
            p.masked_fill_(~seen, -math.inf)
        p = p.sub_(p.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True))
        o = torch.bmm(p.view(c.h, g * n, end), v).view(c.h, g, n, d).permute(2, 0, 1, 3)
        out[at[i]:at[i + 1]] = o.reshape(n, h, d)
    return out


# -------------------------------------------------------------------- calls --

def _plan(s):
    """The call's shape and workspace, made on a state's first pass and kept, as a user's program keeps them."""
    path = os.path.join(os.getcwd(), "odin-infer_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from oi import paged
    case, op = s["case"], s["op"]
    if op == "plan":
        s["plan"] = paged.Paged(8, 128, s["n_pages"], case["page"])
        return
    c = s["c"]
    s["plan"] = paged.Paged(c.h, c.d, c.n, c.p)
    if op == "tokens":
        need = s["plan"].tokens_workspace_bytes(case["heads"], case["seqs"], case["n"])
    elif op == "prompts":
        need = s["plan"].prompts_workspace_bytes(case["heads"], case["seqs"], s["q"].shape[0])
    else:
        return
    s["ws"] = torch.empty(need, dtype=torch.uint8, device=DEV)


def _own(s):
    if "plan" not in s:
        _plan(s)
    case, op, plan = s["case"], s["op"], s["plan"]
    st = torch.cuda.current_stream().cuda_stream
    if op == "plan":
        n, width, rows = case["seqs"], s["width"], s["n_rows"]
        plan.plan(n, s["past"].data_ptr(), s["new"].data_ptr(), s["table"].data_ptr(), width, s["free"].data_ptr(),
                  s["n_free"].data_ptr(), rows, s["lens"].data_ptr(), s["starts"].data_ptr(), s["slots"].data_ptr(),
                  s["pos"].data_ptr(), stream=st)
        # what was taken goes back: requests hold lens slots and keep past of them
        plan.release(n, s["lens"].data_ptr(), s["past"].data_ptr(), s["table"].data_ptr(), width, s["free"].data_ptr(),
                     s["n_free"].data_ptr(), stream=st)
        return s["table"], s["lens"], s["starts"], s["slots"][:rows], s["pos"][:, :rows], s["free"], s["n_free"]
    c, t = s["c"], CODES[case["type"]]
    buf = c.buf.data_ptr()
    if op == "append":
        plan.append(buf, t, s["k"].data_ptr(), s["v"].data_ptr(), s["slots"].numel(), s["slots"].data_ptr(), stream=st)
        return c.k, c.v
    args = (s["lens"].data_ptr(), c.table.data_ptr(), c.width, s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel())
    if op == "tokens":
        plan.tokens(buf, case["heads"], t, s["q"].data_ptr(), case["seqs"], case["n"], *args, stream=st)
    else:
        plan.prompts(buf, case["heads"], t, s["q"].data_ptr(), case["seqs"], s["q"].shape[0], s["starts"].data_ptr(),
                     *args, stream=st)
    return s["out"]


def run(s):
    if own:
        return _own(s)
    op = s["op"]
    return _plain_plan(s) if op == "plan" else _plain_append(s) if op == "append" else _plain_attn(s)


# --------------------------------------------------------------------- work --

def work(case):
    op = case["op"]
    past, new = _lengths(case)
    total = sum(new)
    if op == "plan":
        rows, p = total + case["pad"], case["page"]
        taken = sum(_pages(x + y, p) - _pages(x, p) for x, y in zip(past, new))
        return {"bytes": 16 * case["seqs"] + 16 * rows + 16 * taken, "flops": 8 * rows}
    hk, d, z = case["kv_heads"], case["head_dim"], SIZE[case["type"]]
    if op == "append":
        return {"bytes": 2 * hk * d * total * (z + 2) + 4 * (total + case["pad"]), "flops": 2 * hk * d * total}
    h = case["heads"]
    seen = sum(n * x + n * (n + 1) // 2 for x, n in zip(past, new))
    slots = sum(x + n for x, n in zip(past, new))
    return {"bytes": 4 * hk * d * slots + 2 * total * h * d * z + 4 * _pages(slots, case["page"]),
            "flops": 4 * h * d * seen}


# ------------------------------------------------------- in 64 bits, apart --

def _exact_plan(case, s):
    """Request after request on the host."""
    p, width, rows = case["page"], s["width"], s["n_rows"]
    past, new, free = s["past"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, n_free = s["table"].tolist(), s["n_free"].item()
    lens, starts, slots, pos = [], [0], [-1] * rows, [0] * rows
    wanted = taken = 0
    for i, (a, b) in enumerate(zip(past, new)):
        row0, lens_i = starts[-1], 0
        starts.append(min(rows, row0 + b))
        if sum(new[:i + 1]) <= rows and a + b <= width * p:
            have = -(-a // p)
            more = -(-(a + b) // p) - have
            wanted += more
            if more == 0 or wanted <= n_free:
                for k in range(more):
                    table[i][have + k] = free[n_free - 1 - taken]
                    taken += 1
                for k in range(b):
                    slots[row0 + k] = table[i][(a + k) // p] * p + (a + k) % p
                    pos[row0 + k] = a + k
                lens_i = a + b
        lens.append(lens_i)
    return (_ints(table).view(-1, width), _ints(lens), _ints(starts), _ints(slots), _ints(pos).expand(3, rows), s["free"],
            s["n_free"])


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "plan":
        return _exact_plan(case, s)
    c = s["c"]
    if op == "append":
        k, v = c.k.double(), c.v.double()
        slots = s["slots"].tolist()
        rows = [i for i, x in enumerate(slots) if x >= 0]
        flat = torch.tensor([slots[i] for i in rows], device=DEV)
        for head in range(c.h):
            for which, x in (("k", s["k"]), ("v", s["v"])):
                y = x[rows, head].double().nan_to_num(0.0, TOP, -TOP).clamp(-TOP, TOP)
                for a in range(0, len(rows), 4096):
                    f, z = flat[a:a + 4096], y[a:a + 4096]
                    if which == "k":
                        k[f // c.p, head, f % c.p] = z
                    else:
                        v[f // c.p, head, f % c.p // 8, :, f % 8] = z
        return k, v
    h, d = case["heads"], case["head_dim"]
    g = h // c.h
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    a = 0
    for i, (past, n) in enumerate(zip(s["past"], s["new"])):
        end = past + n
        j = torch.arange(end, device=DEV)
        page, off = c.table[i].long()[j // c.p], j % c.p
        last = past + torch.arange(n, device=DEV)
        for r in range(h):
            k = c.k[page, r // g, off].double()
            v = c.v[page, r // g, off // 8, :, off % 8].double()
            x = (s["q"][a:a + n, r].double() @ k.t()) / math.sqrt(d)
            x[j[None] > last[:, None]] = -math.inf
            out[a:a + n, r] = torch.softmax(x, 1) @ v
        a += n
    return out
