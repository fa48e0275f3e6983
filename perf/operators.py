"""Operators around a decode cache that is kept small: held in 4 bits, and cut to the keys that attention still looks at.

A case is one pass of one of them, on tensors that sit in HBM.  The kinds:

    append    rotary embedding of new q and k and their append to a cache of 4-bit values, then the rows read back
    attend    attention of one or several new positions per sequence over a cache of 4-bit values
    weigh     attention of one new token per sequence that adds every key's weight to a running sum, over a bf16 or a
              4-bit cache
    evict     from those sums, the rows of a bf16 cache that stay, moved together

The 4-bit cache.  A row of 64, 128 or 256 values has a pair of bf16 numbers (scale s, middle z) for each 64 of them, and a
value is z + s (c - 8) with a code c of 0 to 15.  For the group's largest and smallest value, hi and lo:

    z = bf16((hi + lo) / 2 + (hi - lo) / 32)      s = max((hi - z) / 7.5, (z - lo) / 8.5), rounded up to a bf16
    c = 8 + the whole number nearest to (x - z) / s, ties to even, within -8 .. 7      (8 where s is 0)

Codes lie as bytes [batch, kv heads, rows, dim / 2]: with n = dim / 32, byte i n + p holds dims 32 c + 2 i (low bits) and
32 c + 2 i + 1, where c is p with its lowest two bits exchanged (for n = 2: c = p).  The pairs lie as 32-bit words [batch,
kv heads, dim / 64, rows], s in the low half.
"""
import math

import torch

own = False  # False: the plain forms; True: the library's operators


def listed():
    return [
        # one token of one conversation: the smallest call
        {"name": "append_token_b1_gqa_d128", "kind": "append", "batch": 1, "heads": 32, "kv_heads": 8, "seq": 1,
         "max_seq": 4096, "dim": 128},
        # two long prompts
        {"name": "append_prompt_b2_gqa_n4096_d128", "kind": "append", "batch": 2, "heads": 32, "kv_heads": 8, "seq": 4096,
         "max_seq": 8192, "dim": 128},
        # one token of one conversation of ordinary length
        {"name": "attend_b1_gqa_ctx2048_d128", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "new": 1,
         "shortest": 2048, "context": 2048, "max_seq": 4096, "dim": 128},
        # a serving batch of sequences of 512 to 8192 tokens
        {"name": "attend_b64_gqa_ctx8192_d128", "kind": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "new": 1,
         "shortest": 512, "context": 8192, "max_seq": 8192, "dim": 128},
        # a batch of odd lengths on a model without grouped kv heads
        {"name": "attend_b16_h16_ctx3001_d64", "kind": "attend", "batch": 16, "heads": 16, "kv_heads": 16, "new": 1,
         "shortest": 37, "context": 3001, "max_seq": 3011, "dim": 64},
        # sixteen drafted tokens of one sequence over a long cache
        {"name": "attend_b1_gqa_new16_ctx8192_d128", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "new": 16,
         "shortest": 8192, "context": 8192, "max_seq": 8192, "dim": 128},
        # the running sums of one long conversation
        {"name": "weigh_b1_gqa_ctx8192_d128", "kind": "weigh", "batch": 1, "heads": 32, "kv_heads": 8, "cache": "bf16",
         "shortest": 8192, "context": 8192, "max_seq": 8192, "dim": 128},
        # ... of a batch on a model of few, wide heads
        {"name": "weigh_b16_gqa_ctx4000_d256", "kind": "weigh", "batch": 16, "heads": 16, "kv_heads": 2, "cache": "bf16",
         "shortest": 1000, "context": 4000, "max_seq": 4096, "dim": 256},
        # ... and of a serving batch whose cache is held in 4 bits
        {"name": "weigh_q4_b32_gqa_ctx4096_d128", "kind": "weigh", "batch": 32, "heads": 32, "kv_heads": 8, "cache": "q4",
         "shortest": 300, "context": 4096, "max_seq": 4096, "dim": 128},
        # a long prompt cut to a quarter
        {"name": "evict_b1_gqa_ctx8192_to_2048_d128", "kind": "evict", "batch": 1, "kv_heads": 8, "shortest": 8192,
         "context": 8192, "max_seq": 8192, "budget": 2048, "recent": 256, "dim": 128},
        # a serving batch of which some sequences are short enough to stay whole
        {"name": "evict_b32_gqa_ctx4096_to_1500_d128", "kind": "evict", "batch": 32, "kv_heads": 8, "shortest": 300,
         "context": 4096, "max_seq": 4096, "budget": 1500, "recent": 100, "dim": 128},
    ]


# ---- drawn cases ------------------------------------------------------------------------------------------------


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm; odd ones as likely as even ones."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_BYTES = 3.0e8  # of a drawn case: below the largest listed one's


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "attend", "weigh", "weigh", "evict"))
    heads, kv_heads = rng.choice(((8, 8), (16, 16), (32, 8), (32, 8), (12, 12), (16, 2), (40, 8), (28, 4), (32, 2), (34, 2)))
    case = {"kind": kind, "batch": _log(rng, 1, 64), "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128, 256))}
    if kind != "evict":
        case["heads"] = heads
    if kind == "append":
        case["seq"] = rng.choice((1, 1, _log(rng, 2, 8192)))
        case["max_seq"] = case["seq"] + _log(rng, 1, 4096)
    else:
        context = _log(rng, 1, 16384)
        case.update(shortest=max(1, context // rng.randint(1, 16)), context=context, max_seq=context + _log(rng, 1, 512))
        if kind == "attend":
            case["new"] = rng.choice((1, 1, 1, _log(rng, 2, 64)))
        elif kind == "weigh":
            case["cache"] = rng.choice(("bf16", "q4"))
        else:
            case["budget"] = _log(rng, 1, context)
            case["recent"] = rng.choice((0, _log(rng, 1, case["budget"])))
    while work(case)["bytes"] > _MOST_BYTES or case["batch"] * case["kv_heads"] * case["max_seq"] * case["dim"] > 1 << 29:
        if case["batch"] > 1:
            case["batch"] //= 2
        else:
            case["seq"] = case["seq"] // 2
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------


def _lengths(case):
    """The batch's lengths, evenly spread from the shortest to the longest."""
    b, lo, hi = case["batch"], case["shortest"], case["context"]
    return [hi] if b == 1 else [lo + (hi - lo) * i // (b - 1) for i in range(b)]


class _Tables:
    """cos and sin of the rotary embedding on the device, [positions, dim / 2] of f32."""

    def __init__(self, dim, max_seq, device):
        self.max_seq = max_seq
        theta = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        angle = torch.arange(max_seq, dtype=torch.float64)[:, None] * theta[None, :]
        self.cos, self.sin = angle.cos().float().to(device), angle.sin().float().to(device)

    def device_tables(self):
        return self.cos, self.sin


def _byte_order(dim):
    """Dims of the two values of each byte of a row, [dim / 2, 2]."""
    n = dim // 32
    at = torch.arange(dim // 2)
    i, p = at // n, at % n
    c = p if n == 2 else (p & ~3) | (p & 1) << 1 | (p >> 1 & 1)
    return torch.stack((32 * c + 2 * i, 32 * c + 2 * i + 1), -1)


def _quantise(x):
    """x [.., rows, dim] -> codes [.., rows, dim / 2] of bytes and pairs [.., dim / 64, rows] of 32-bit words."""
    d = x.shape[-1]
    g = x.float().unflatten(-1, (d // 64, 64))
    hi, lo = g.amax(-1), g.amin(-1)
    z = ((hi + lo) * 0.5 + (hi - lo) * (1 / 32)).bfloat16().float()
    # (divided by tensors: a division by a number may be a product with its rounded inverse)
    s = torch.maximum((hi - z) / torch.full_like(z, 7.5), (z - lo) / torch.full_like(z, 8.5))
    s = ((s.view(torch.int32) + 0xffff) & -65536).view(torch.float32)
    c = torch.round((g - z[..., None]).double() / s[..., None].double()).clamp(-8, 7)
    c = torch.where(s[..., None] == 0, 0.0, c).flatten(-2).to(torch.int32) + 8
    two = c[..., _byte_order(d).to(c.device)]
    codes = (two[..., 0] | two[..., 1] << 4).to(torch.uint8)
    pairs = (s.view(torch.int32) >> 16 & 0xffff) | (z.view(torch.int32) & -65536)
    return codes, pairs.transpose(-1, -2).contiguous()


def _values(codes, pairs):
    """What a 4-bit cache stands for, [.., rows, dim]."""
    d = 2 * codes.shape[-1]
    c = torch.empty(*codes.shape[:-1], d, device=codes.device)
    order = _byte_order(d).to(codes.device)
    c[..., order[:, 0]] = (codes & 15).float()
    c[..., order[:, 1]] = (codes >> 4).float()
    s = (pairs << 16).view(torch.float32).transpose(-1, -2)
    z = (pairs & -65536).view(torch.float32).transpose(-1, -2)
    return (z[..., None] + s[..., None] * (c.unflatten(-1, (d // 64, 64)) - 8)).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def bf16(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    kind, b, hkv, d, n = case["kind"], case["batch"], case["kv_heads"], case["dim"], case["max_seq"]
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}

    def cache(rows):
        # keys and values as layers leave them: a few channels of a head are much larger than the others
        wide = 1 + 4 * (torch.rand(hkv, 1, d, generator=gen, device="cuda") < 0.03).to(torch.bfloat16)
        return bf16(b, hkv, rows, d) * wide

    if kind == "append":
        new = case["seq"]
        s["q"], s["k_in"], s["v_in"] = bf16(b, case["heads"], new, d), cache(new), cache(new)
        s["q_out"] = torch.empty_like(s["q"])
        s["rope"] = _Tables(d, n, "cuda")
        # sequences that have reached different positions
        at = [0 if b == 1 and new > 1 else (n - new) * (i + 1) // b for i in range(b)]
        s["positions"] = torch.tensor(at, dtype=torch.int32, device="cuda")[torch.randperm(b, generator=gen, device="cuda")].contiguous()
        for x in ("k", "v"):
            s[x + "_codes"] = torch.zeros(b, hkv, n, d // 2, dtype=torch.uint8, device="cuda")
            s[x + "_pairs"] = torch.zeros(b, hkv, d // 64, n, dtype=torch.int32, device="cuda")
            s[x + "_rows"] = torch.empty(b, hkv, new, d, dtype=torch.bfloat16, device="cuda")
        return s
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    s["lens"] = lens[torch.randperm(b, generator=gen, device="cuda")].contiguous()
    if kind == "evict":
        s["k"], s["v"] = bf16(b, hkv, n, d), bf16(b, hkv, n, d)
        # sums of attention weights: most keys hardly looked at, a few again and again; every eighth key never
        w = torch.exp(2 * torch.randn(b, hkv, n, generator=gen, device="cuda"))
        s["weights"] = torch.where(torch.rand(b, hkv, n, generator=gen, device="cuda") < 0.125, 0.0, w)
        s["slots"] = torch.arange(n, dtype=torch.int32, device="cuda").expand(b, hkv, n).contiguous()
        s["weights_out"], s["slots_out"] = torch.zeros_like(s["weights"]), torch.zeros_like(s["slots"])
        s["new_lens"] = torch.zeros_like(s["lens"])
        return s
    q4 = kind == "attend" or case["cache"] == "q4"
    s["q"] = bf16(b, case.get("new", 1), case["heads"], d)
    s["out"] = torch.empty_like(s["q"])
    for x in ("k", "v"):
        rows = cache(n)
        if q4:
            codes = torch.empty(b, hkv, n, d // 2, dtype=torch.uint8, device="cuda")
            pairs = torch.empty(b, hkv, d // 64, n, dtype=torch.int32, device="cuda")
            for i in range(b):
                codes[i], pairs[i] = _quantise(rows[i])
            s[x + "_codes"], s[x + "_pairs"] = codes, pairs
        else:
            s[x] = rows
    if kind == "weigh":
        s["weights"] = torch.rand(b, hkv, n, generator=gen, device="cuda")
        s["weights_out"] = torch.zeros_like(s["weights"])
    return s


# ---- one pass, the plain forms ------------------------------------------------------------------------------------


def _rotate(x, cos, sin):
    """Half-split rotary embedding of [b, heads, seq, dim] by tables [b, 1, seq, dim / 2], in 32 bits."""
    a, c = x.float().chunk(2, -1)
    return torch.cat((a * cos - c * sin, c * cos + a * sin), -1)


def _plain_append(s):
    new, n = s["case"]["seq"], s["case"]["max_seq"]
    at = s["positions"].long()[:, None] + torch.arange(new, device="cuda")
    cos, sin = (t[at][:, None] for t in s["rope"].device_tables())
    s["q_out"].copy_(_rotate(s["q"], cos, sin))
    for x, rows in (("k", _rotate(s["k_in"], cos, sin)), ("v", s["v_in"].float())):
        codes, pairs = _quantise(rows)
        s[x + "_codes"].scatter_(2, at[:, None, :, None].expand_as(codes), codes)
        s[x + "_pairs"].scatter_(3, at[:, None, None, :].expand_as(pairs), pairs)
        s[x + "_rows"].copy_(_values(codes, pairs))
    return {"q": s["q_out"], "k_rows": s["k_rows"], "v_rows": s["v_rows"]}


def _plain_attention(s, k, v):
    """Values [b, new, heads, dim] and weights [b, kv heads, new * group, keys], in 32 bits."""
    q, lens = s["q"].float(), s["lens"]
    b, new, h, d = q.shape
    hkv, n = k.shape[1], k.shape[2]
    q = q.reshape(b, new, hkv, h // hkv, d).transpose(1, 2).reshape(b, hkv, new * (h // hkv), d)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)
    end = lens[:, None] - new + 1 + torch.arange(new, device="cuda").repeat_interleave(h // hkv)  # keys that a row sees
    x = torch.where(torch.arange(n, device="cuda") < end[:, None, :, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, v).reshape(b, hkv, new, h // hkv, d).transpose(1, 2).reshape(b, new, h, d)
    return out, p


def _plain_cache(s):
    if "k" in s:
        return s["k"].float(), s["v"].float()
    return _values(s["k_codes"], s["k_pairs"]), _values(s["v_codes"], s["v_pairs"])


def _plain_evict(s):
    c, lens = s["case"], s["lens"].long()
    b, hkv, n = s["weights"].shape
    budget = c["budget"]
    slot = torch.arange(n, device="cuda").expand(b, hkv, n)
    there = slot < lens[:, None, None]
    newest = torch.where(there, s["slots"], -1).amax(-1, keepdim=True)
    w = torch.where(torch.isnan(s["weights"]), -math.inf, s["weights"])
    w = torch.where(s["slots"] > newest - c["recent"], math.inf, w)
    w = torch.where(there, w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices  # equal sums: the lower slot first
    rank = torch.empty_like(order).scatter_(-1, order, slot.contiguous())
    new_lens = lens.clamp(max=budget)
    keep = rank < new_lens[:, None, None]
    # the i-th free slot below the new length takes the i-th row that is kept above it
    free, moves = ~keep & (slot < new_lens[:, None, None]), keep & (slot >= new_lens[:, None, None])
    taken = torch.zeros(b, hkv, n + 1, dtype=torch.int64, device="cuda")
    taken.scatter_(-1, torch.where(moves, moves.cumsum(-1) - 1, n), slot.contiguous())
    source = torch.where(free, taken.gather(-1, (free.cumsum(-1) - 1).clamp(min=0)), slot)[..., :budget]
    inside = (slot < new_lens[:, None, None])[..., :budget]
    wide = source[..., None].expand(b, hkv, budget, c["dim"])
    for x in ("k", "v"):
        s[x][:, :, :budget] = torch.where(inside[..., None], s[x].gather(2, wide), s[x][:, :, :budget])
    for x in ("weights", "slots"):
        at = s[x + "_out"][..., :budget]
        at.copy_(torch.where(inside, s[x].gather(-1, source), at))
    s["new_lens"].copy_(new_lens)
    return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "slots": s["slots_out"], "lens": s["new_lens"]}


# ---- one pass -----------------------------------------------------------------------------------------------------


def _workspace(s, size):
    """Scratch that a program keeps from call to call."""
    if "ws" not in s:
        s["ws_bytes"] = max(256, size())
        s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device="cuda")
    return s["ws"], s["ws_bytes"]


def _own(s):
    from rustorch_amd import LlmKernels as K, Q4Rows

    c, stream = s["case"], s["stream"]
    b, hkv, d, n = c["batch"], c["kv_heads"], c["dim"], c["max_seq"]
    if c["kind"] == "evict":
        ws = _workspace(s, lambda: K.kv_evict_workspace_bytes(b, hkv, n, c["budget"]))
        K.kv_evict_bf16(stream, s["k"], s["v"], s["weights"], s["slots"], s["weights_out"], s["slots_out"], s["lens"],
                        s["new_lens"], b, hkv, d, n, c["budget"], c["recent"], *ws)
        return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "slots": s["slots_out"], "lens": s["new_lens"]}
    h = c["heads"]
    if "k" in s:
        k, v = s["k"], s["v"]
    else:
        k, v = Q4Rows(s["k_codes"], s["k_pairs"]), Q4Rows(s["v_codes"], s["v_pairs"])
    if c["kind"] == "append":
        K.qk_norm_rope_kv_append_q4(stream, s["q"], s["q_out"], s["k_in"], s["v_in"], k, v, s["positions"], s["rope"], b, h,
                                    hkv, d, n, seq=c["seq"])
        K.kv_cache_read_q4(stream, k, s["k_rows"], b, hkv, d, n, s["positions"], c["seq"])
        K.kv_cache_read_q4(stream, v, s["v_rows"], b, hkv, d, n, s["positions"], c["seq"])
        return {"q": s["q_out"], "k_rows": s["k_rows"], "v_rows": s["v_rows"]}
    if c["kind"] == "attend":
        ws = _workspace(s, lambda: K.gqa_decode_q4_workspace_bytes(b, c["new"], h, hkv, d, n))
        K.gqa_decode_q4(stream, s["q"], k, v, s["out"], s["lens"], b, c["new"], h, hkv, d, n, *ws)
        return s["out"]
    ws = _workspace(s, lambda: K.gqa_decode_weights_workspace_bytes(b, h, hkv, d, n))
    call = K.gqa_decode_weights_q4 if c["cache"] == "q4" else K.gqa_decode_weights_bf16
    call(stream, s["q"], k, v, s["out"], s["weights"], s["weights_out"], s["lens"], b, h, hkv, d, n, *ws)
    return {"out": s["out"], "weights": s["weights_out"]}


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "append":
        return _plain_append(s)
    if kind == "evict":
        return _plain_evict(s)
    out, p = _plain_attention(s, *_plain_cache(s))
    s["out"].copy_(out)
    if kind == "attend":
        return s["out"]
    b, hkv, _, n = p.shape
    there = torch.arange(n, device="cuda") < s["lens"][:, None, None]
    s["weights_out"].copy_(torch.where(there, s["weights"] + p.sum(2), s["weights_out"]))
    return {"out": s["out"], "weights": s["weights_out"]}


# ---- the same from the definition, in 64 bits -----------------------------------------------------------------------


def _exact_rows(x):
    """Rows of f64 as the 4-bit cache gives them back."""
    g = x.reshape(*x.shape[:-1], -1, 64)
    hi, lo = g.max(-1, keepdim=True).values, g.min(-1, keepdim=True).values
    z = ((hi + lo) / 2 + (hi - lo) / 32).to(torch.bfloat16).double()
    s = torch.maximum((hi - z) / 7.5, (z - lo) / 8.5)
    down = s.to(torch.bfloat16)
    step = torch.nextafter(down.float(), torch.full_like(down.float(), math.inf))  # (only tells which way it was rounded)
    up = torch.where(down.double() < s, ((step.view(torch.int32) >> 16) + 1 << 16).view(torch.float32).double(), down.double())
    c = torch.round((g - z) / torch.where(up == 0, 1.0, up)).clamp(-8, 7)
    return (z + up * c).reshape(x.shape)


def _exact_cache(codes, pairs):
    """Rows [n, dim] of f64 that the codes [n, dim / 2] and pairs [dim / 64, n] of one head stand for."""
    rows, half = codes.shape
    n = half // 16
    x = torch.stack((codes & 15, codes >> 4), -1).double().view(rows, 16, n, 2)
    x = x[:, :, [0, 1] if n == 2 else [4 * (p // 4) + (0, 2, 1, 3)[p % 4] for p in range(n)]]
    x = x.permute(0, 2, 1, 3).reshape(rows, n // 2, 64)
    sz = pairs.contiguous().view(torch.bfloat16).double().view(n // 2, rows, 2).transpose(0, 1)
    return (sz[..., 1:] + sz[..., :1] * (x - 8)).reshape(rows, -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind, b, hkv = case["kind"], case["batch"], case["kv_heads"]
    if kind == "evict":
        return None  # a selection: whole values, and rows as they are
    if kind == "append":
        new, half = case["seq"], case["dim"] // 2
        cos, sin = (t.double() for t in s["rope"].device_tables())
        got = {x: [] for x in ("q", "k_rows", "v_rows")}
        for i, p in enumerate(s["positions"].tolist()):
            turned = []
            for x in (s["q"][i].double(), s["k_in"][i].double()):
                y = torch.empty_like(x)
                y[..., :half] = x[..., :half] * cos[p:p + new] - x[..., half:] * sin[p:p + new]
                y[..., half:] = x[..., half:] * cos[p:p + new] + x[..., :half] * sin[p:p + new]
                turned.append(y)
            got["q"].append(turned[0])
            got["k_rows"].append(_exact_rows(turned[1]))
            got["v_rows"].append(_exact_rows(s["v_in"][i].double()))
        return {x: torch.stack(y) for x, y in got.items()}
    new, h, d, n = case.get("new", 1), case["heads"], case["dim"], case["max_seq"]
    out = torch.zeros(b, new, h, d, dtype=torch.float64, device="cuda")
    weights = torch.zeros(b, hkv, n, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s["lens"].tolist()):
        for j in range(hkv):
            if "k" in s:
                k, v = s["k"][i, j, :length].double(), s["v"][i, j, :length].double()
            else:
                k, v = (_exact_cache(s[x + "_codes"][i, j, :length], s[x + "_pairs"][i, j, :, :length]) for x in ("k", "v"))
            heads = slice(j * (h // hkv), (j + 1) * (h // hkv))
            x = s["q"][i, :, heads].double() @ k.T / math.sqrt(d)  # [new, heads of the group, keys]
            for t in range(new):
                x[t, :, max(0, length - new + t + 1):] = -math.inf
            p = torch.softmax(x, -1).nan_to_num(0.0)  # a position that sees no key: zeros
            out[i, :, heads] = p @ v
            if kind == "weigh":
                weights[i, j, :length] = s["weights"][i, j, :length].double() + p.sum((0, 1))
    return out if kind == "attend" else {"out": out, "weights": weights}


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    kind, b, hkv, d = case["kind"], case["batch"], case["kv_heads"], case["dim"]
    row4 = d // 2 + d // 16  # bytes of a row of a 4-bit cache
    if kind == "append":  # q in and out, k and v in, their cache rows out and in again, those as bf16 out; the table rows
        n, h = case["seq"], case["heads"]
        return {"bytes": b * n * (4 * h * d + hkv * (8 * d + 4 * row4)) + 4 * n * d, "flops": b * n * d * (3 * h + 20 * hkv)}
    lens = _lengths(case)
    if kind == "evict":
        # sums and positions in; of a sequence above the budget the rows that move, in and out; below, sums and positions out
        total = 0.0
        for n in lens:
            total += 8 * n + 8 * min(n, case["budget"])
            if n > case["budget"]:
                rest = n - min(case["recent"], case["budget"])
                free = case["budget"] - min(case["recent"], case["budget"])
                # the newest rows lie last; of the others, which are kept by chance, as many move as are kept behind the budget
                late = max(0, rest - case["budget"])
                total += 8 * d * ((n - max(rest, case["budget"])) + (free * late / rest if rest else 0))
        return {"bytes": hkv * total, "flops": 0}
    h, new = case["heads"], case.get("new", 1)
    keys = sum(lens)
    pairs = sum(max(0, n - new + t + 1) for n in lens for t in range(new))
    row = row4 if kind == "attend" or case["cache"] == "q4" else 2 * d
    sums = 8 * hkv * keys if kind == "weigh" else 0
    return {"bytes": 2 * hkv * keys * row + 4 * b * new * h * d + sums, "flops": 4 * h * d * pairs}
