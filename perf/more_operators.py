"""Operators of a server that holds many requests side by side: prompts packed one behind the other, and a cache in pages.

A case is one pass of one of them, on tensors that sit in HBM.  The kinds:

    append    RMSNorm and rotary embedding of packed new q and k, and their append, with v, to a cache in pages; with one
              position a token, or with one on each of three axes (time, height, width)
    prompt    causal attention of whole prompts packed one behind the other
    decode    attention of one new token per sequence over a cache in pages; `shared` leading keys, 0 for none, are those of a
              prefix that all sequences have in common, in the same pages

The cache.  K and V are [pages, kv heads, rows of a page, dim]; row r of sequence b lies in page table[b, r // rows], there
in row r % rows.  An entry of the table that is no page (-1) stands for rows that are not there.
"""
import math

import torch

own = False  # False: the plain forms; True: the library's operators


def listed():
    return [
        # one token of one conversation: the smallest call
        {"name": "append_token_b1_gqa_d128", "kind": "append", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "prompt": False, "shortest": 2048, "longest": 2048, "norm": True, "axes": False},
        # four long prompts of different lengths
        {"name": "append_prompts_b4_gqa_n4096_d128", "kind": "append", "batch": 4, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "prompt": True, "shortest": 1501, "longest": 4096, "norm": True, "axes": False},
        # a decode step of a batch whose prompts had images in them
        {"name": "append_axes_step_b64_gqa_d128", "kind": "append", "batch": 64, "heads": 28, "kv_heads": 4, "dim": 128,
         "page": 16, "prompt": False, "shortest": 300, "longest": 4096, "norm": False, "axes": True},
        # prompts of text and images
        {"name": "append_axes_prompts_b6_h16_n2000_d64", "kind": "append", "batch": 6, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 32, "prompt": True, "shortest": 333, "longest": 2000, "norm": False, "axes": True},
        # a few short prompts
        {"name": "prompt_b3_h16_n300_d64", "kind": "prompt", "batch": 3, "heads": 16, "kv_heads": 16, "dim": 64,
         "shortest": 77, "longest": 300},
        # a serving batch of ordinary prompts, odd lengths
        {"name": "prompt_b16_gqa_n2000_d128", "kind": "prompt", "batch": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "shortest": 101, "longest": 2000},
        # long documents
        {"name": "prompt_b3_gqa_n8192_d128", "kind": "prompt", "batch": 3, "heads": 32, "kv_heads": 8, "dim": 128,
         "shortest": 1300, "longest": 8192},
        # few, wide heads
        {"name": "prompt_b8_gqa_n1024_d256", "kind": "prompt", "batch": 8, "heads": 16, "kv_heads": 2, "dim": 256,
         "shortest": 64, "longest": 1024},
        # one token of one conversation of ordinary length
        {"name": "decode_b1_gqa_ctx2048_d128", "kind": "decode", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "shared": 0, "shortest": 2048, "longest": 2048},
        # a serving batch of sequences of 512 to 8192 tokens that have nothing in common
        {"name": "decode_b64_gqa_ctx8192_d128", "kind": "decode", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "shared": 0, "shortest": 512, "longest": 8192},
        # 64 conversations behind one long document
        {"name": "shared_b64_gqa_8192_own512_d128", "kind": "decode", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "shared": 8192, "shortest": 8200, "longest": 8704},
        # 24 samples of one prompt of odd length, on a model without grouped kv heads
        {"name": "shared_b24_h16_1001_own2000_d64", "kind": "decode", "batch": 24, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 16, "shared": 1001, "shortest": 1002, "longest": 3001},
    ]


# ---- drawn cases ------------------------------------------------------------------------------------------------


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm; odd ones as likely as even ones."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST = {"bytes": 4.0e8, "flops": 4.0e11}  # of a drawn case: below the largest listed one's


def draw(rng):
    kind = rng.choice(("append", "append", "prompt", "prompt", "decode", "decode", "decode"))
    heads, kv_heads = rng.choice(((8, 8), (16, 16), (32, 8), (32, 8), (12, 12), (16, 2), (40, 8), (28, 4), (32, 2), (34, 2), (20, 1)))
    case = {"kind": kind, "batch": _log(rng, 1, 64), "heads": heads, "kv_heads": kv_heads, "dim": rng.choice((64, 80, 96, 128, 128, 256))}
    if kind != "prompt":
        case["page"] = rng.choice((16, 16, 32, 64, 128, 256))
    case["longest"] = _log(rng, 1, 8192 if kind == "prompt" else 16384)
    case["shortest"] = max(1, case["longest"] // rng.randint(1, 16))
    if kind == "append":
        case.update(prompt=rng.choice((False, True)), norm=rng.choice((False, True)), axes=rng.choice((False, False, True)))
    elif kind == "decode":
        case["shared"] = rng.choice((0, rng.randint(1, case["shortest"]), case["shortest"]))
    while any(work(case)[x] > _MOST[x] for x in _MOST) or _plain_size(case) > 3e9:
        if case["batch"] > 1:
            case["batch"] //= 2
        else:
            case["longest"] //= 2
            case["shortest"] = min(case["shortest"], case["longest"])
            case.update({"shared": min(case["shared"], case["shortest"])} if kind == "decode" else {})
    return case


def _plain_size(case):
    """Values that the plain form holds of one kind."""
    if case["kind"] == "append":
        return 0
    b, n = case["batch"], case["longest"]
    return b * n * (case["heads"] * n if case["kind"] == "prompt" else 2 * case["kv_heads"] * case["dim"])


# ---- inputs -----------------------------------------------------------------------------------------------------


def _lengths(case):
    """The batch's lengths, evenly spread from the shortest to the longest."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
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


def _sections(dim):
    """Pairs of a head that turn with each of the three axes: a quarter, and three eighths twice."""
    half = dim // 2
    time = half // 4
    height = (half - time) // 2
    return (time, height, half - time - height)


def _axis_positions(rows):
    """[3, tokens] of rows' positions on the axes, for sequences of a text of 32 tokens and then images of 16 x 16 patches."""
    image, j = (rows - 32).clamp(min=0) // 256, (rows - 32).clamp(min=0) % 256
    first = 32 + 16 * image
    text = rows < 32
    return torch.stack([torch.where(text, rows, x) for x in (first, first + j // 16, first + j % 16)]).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def bf16(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    kind, b, h, hkv, d = (case[x] for x in ("kind", "batch", "heads", "kv_heads", "dim"))
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    # the batch's lengths, in any order
    lens = torch.tensor(_lengths(case), dtype=torch.int64)
    lens = lens[torch.randperm(b, generator=torch.Generator().manual_seed(seed))]
    starts = torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0))).to(device="cuda", dtype=torch.int32)
    # keys and values as layers leave them: a few channels of a head are much larger than the others
    wide = 1 + 4 * (torch.rand(hkv, 1, d, generator=gen, device="cuda") < 0.03).to(torch.bfloat16)

    if kind == "prompt":
        t = int(lens.sum())
        s.update(tokens=t, starts=starts, q=bf16(t, h, d), k=bf16(t, hkv, d) * wide[:, 0], v=bf16(t, hkv, d))
        s["out"] = torch.empty_like(s["q"])
        return s

    page, shared = case["page"], case.get("shared", 0)
    table_pages = -(-case["longest"] // page) + 1
    need = (lens + page - 1) // page  # pages that each sequence has
    common = shared // page  # whole pages of the prefix: the same for all.  (Of a page that ends behind it everybody has a copy.)
    col = torch.arange(table_pages)
    number = torch.where(col < common, col, common + (need - common).clamp(min=0).cumsum(0)[:, None] - (need - common).clamp(min=0)[:, None] + col - common)
    n_pages = common + int((need - common).clamp(min=0).sum()) + 3
    table = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed + 1))[number.clamp(max=n_pages - 1)]
    s["table"] = torch.where(col < need[:, None], table, -1).to(device="cuda", dtype=torch.int32).contiguous()
    s["n_pages"], s["table_pages"], s["lens"] = n_pages, table_pages, lens.to(device="cuda", dtype=torch.int32)
    s["k_pages"], s["v_pages"] = bf16(n_pages, hkv, page, d) * wide, bf16(n_pages, hkv, page, d)
    if kind == "decode":
        if shared % page:
            # the prefix's last rows, in everybody's own page
            for x in ("k_pages", "v_pages"):
                own_page = s["table"][:, common].long()
                s[x][own_page, :, :shared % page] = s[x][own_page[0], :, :shared % page].clone()
        s["q"] = bf16(b, h, d)
        s["out"] = torch.empty_like(s["q"])
        return s

    # append: whole prompts, or the last token of each sequence
    t = int(lens.sum()) if case["prompt"] else b
    s["tokens"], s["starts"] = t, starts if case["prompt"] else None
    s["positions"] = torch.zeros_like(s["lens"]) if case["prompt"] else s["lens"] - 1
    s["rope"] = _Tables(d, case["longest"], "cuda")
    s["q"], s["k_in"], s["v_in"] = bf16(t, h, d), bf16(t, hkv, d) * wide[:, 0], bf16(t, hkv, d)
    s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k_in"])
    for x in ("q_gamma", "k_gamma"):
        s[x] = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda") if case["norm"] else None
    s["axes"] = _axis_positions(_token_rows(s)[1]) if case["axes"] else None
    return s


# ---- one pass, the plain forms ------------------------------------------------------------------------------------


def _token_rows(s):
    """Of every packed token its sequence and its row there."""
    t = torch.arange(s["tokens"], device="cuda")
    if s["starts"] is None:
        return t, s["positions"].long()
    b = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    return b, s["positions"].long()[b] + t - s["starts"].long()[b]


def _norm(x, gamma):
    x = x.float()
    if gamma is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma


def _rotate(x, cos, sin):
    """Half-split rotary embedding of [tokens, heads, dim] by [tokens, 1, dim / 2], in 32 bits."""
    a, c = x.chunk(2, -1)
    return torch.cat((a * cos - c * sin, c * cos + a * sin), -1)


def _plain_append(s):
    d = s["case"]["dim"]
    b, row = _token_rows(s)
    cos, sin = s["rope"].device_tables()
    if s["axes"] is None:
        cos, sin = cos[row], sin[row]
    else:
        sections = torch.tensor(_sections(d), device="cuda")
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), sections, output_size=d // 2)
        at, pair = s["axes"].long()[axis].T, torch.arange(d // 2, device="cuda")
        cos, sin = cos[at, pair], sin[at, pair]
    s["q_out"].copy_(_rotate(_norm(s["q"], s["q_gamma"]), cos[:, None], sin[:, None]))
    s["k_out"].copy_(_rotate(_norm(s["k_in"], s["k_gamma"]), cos[:, None], sin[:, None]))
    page = s["case"]["page"]
    at = s["table"].long()[b, row // page]
    s["k_pages"][at, :, row % page] = s["k_out"]
    s["v_pages"][at, :, row % page] = s["v_in"]
    return {"q": s["q_out"], "k": s["k_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _softmax(x):
    """Over the last dimension; a row of -infinity gives zeros."""
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = x.sum(-1, keepdim=True)
    return x / torch.where(total == 0, 1.0, total)


def _plain_prompt(s):
    c, starts = s["case"], s["starts"].long()
    b, h, hkv, d, n = (c[x] for x in ("batch", "heads", "kv_heads", "dim", "longest"))
    at = torch.arange(n, device="cuda")
    rows = (starts[:-1, None] + at).clamp(max=s["tokens"] - 1)  # [b, n]: padded to the longest
    q, k, v = (s[x][rows].float().transpose(1, 2) for x in ("q", "k", "v"))
    x = torch.matmul(q.reshape(b, hkv, h // hkv * n, d), k.transpose(-1, -2)).reshape(b, hkv, h // hkv, n, n)
    x = torch.where(at[:, None] >= at, x / math.sqrt(d), -math.inf)
    out = torch.matmul(_softmax(x).reshape(b, hkv, h // hkv * n, n), v).reshape(b, h, n, d)
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(starts[1:], t, right=True)
    s["out"].copy_(out[seq, :, t - starts[seq]])
    return s["out"]


def _plain_decode(s):
    c, lens = s["case"], s["lens"]
    b, h, hkv, d, n = (c[x] for x in ("batch", "heads", "kv_heads", "dim", "longest"))
    pages = -(-n // c["page"])
    k, v = (s[x][s["table"][:, :pages].long().clamp(min=0)].transpose(1, 2).reshape(b, hkv, -1, d)[:, :, :n].float() for x in ("k_pages", "v_pages"))
    x = torch.matmul(s["q"].float().reshape(b, hkv, h // hkv, d), k.transpose(-1, -2)) / math.sqrt(d)
    x = torch.where(torch.arange(n, device="cuda") < lens[:, None, None, None], x, -math.inf)
    s["out"].copy_(torch.matmul(_softmax(x), v).reshape(b, h, d))
    return s["out"]


# ---- one pass -----------------------------------------------------------------------------------------------------


def _own(s):
    import rustorch_amd as ra

    c, stream, K = s["case"], s["stream"], ra.LlmKernels
    b, h, hkv, d = (c[x] for x in ("batch", "heads", "kv_heads", "dim"))
    if c["kind"] == "prompt":
        shape = ra.AttentionShape.new(b, h, s["tokens"], d)
        ra.flash_forward_packed_bf16_dev(shape, s["q"], s["k"], s["v"], s["starts"], s["out"], n_kv_heads=hkv, stream=stream)
        return s["out"]
    pages = ra.KVPages(s["k_pages"], s["v_pages"], s["n_pages"], c["page"])
    if c["kind"] == "append":
        K.qk_norm_rope_kv_append_paged_bf16(stream, s["q"], s["q_out"], s["k_in"], s["v_in"], pages, s["table"], s["table_pages"],
                                            s["positions"], s["rope"], s["tokens"], b, h, hkv, d, starts=s["starts"],
                                            k_out=s["k_out"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=1e-6,
                                            axis_positions=s["axes"], sections=_sections(d) if c["axes"] else None)
        return {"q": s["q_out"], "k": s["k_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if "ws" not in s:  # scratch that a program keeps from call to call
        s["ws_bytes"] = max(256, K.gqa_decode_paged_workspace_bytes(b, h, hkv, d, c["page"], s["table_pages"]))
        s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device="cuda")
    K.gqa_decode_paged_bf16(stream, s["q"], pages, s["out"], s["table"], s["table_pages"], s["lens"], b, h, hkv, d, s["ws"],
                            s["ws_bytes"], shared_len=c["shared"])
    return s["out"]


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    return _plain_append(s) if kind == "append" else _plain_prompt(s) if kind == "prompt" else _plain_decode(s)


# ---- the same from the definition, in 64 bits -----------------------------------------------------------------------


def _exact_rows(x, gamma, angle_cos, angle_sin):
    """[heads, dim] f64 rows of one token, normed and turned pair by pair."""
    half = x.shape[-1] // 2
    if gamma is not None:
        x = x * gamma.double() * (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).rsqrt()
    y = torch.empty_like(x)
    y[..., :half] = x[..., :half] * angle_cos - x[..., half:] * angle_sin
    y[..., half:] = x[..., half:] * angle_cos + x[..., :half] * angle_sin
    return y


def exact(case, seed):
    s = prepare(case, seed)
    kind, b, h, hkv, d = (case[x] for x in ("kind", "batch", "heads", "kv_heads", "dim"))
    g = h // hkv
    if kind == "append":
        cos, sin = (x.double() for x in s["rope"].device_tables())
        t = {"q": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), "k": torch.empty(s["k_in"].shape, dtype=torch.float64, device="cuda"),
             "k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        first = s["starts"].tolist() if case["prompt"] else list(range(b + 1))
        ends = [sum(_sections(d)[:i + 1]) for i in range(3)]
        for i in range(b):
            of, n, row0 = slice(first[i], first[i + 1]), first[i + 1] - first[i], int(s["positions"][i])
            if case["axes"]:
                c, z = (torch.cat([x[s["axes"][a, of].long(), e0:e1] for a, (e0, e1) in enumerate(zip([0] + ends, ends))], -1) for x in (cos, sin))
            else:
                c, z = cos[row0:row0 + n], sin[row0:row0 + n]
            t["q"][of] = _exact_rows(s["q"][of].double(), s["q_gamma"], c[:, None], z[:, None])
            t["k"][of] = _exact_rows(s["k_in"][of].double(), s["k_gamma"], c[:, None], z[:, None])
            for p in range(row0 // case["page"], (row0 + n - 1) // case["page"] + 1):
                lo, hi = max(row0, p * case["page"]), min(row0 + n, (p + 1) * case["page"])
                at, tok = int(s["table"][i, p]), slice(first[i] + lo - row0, first[i] + hi - row0)
                rows = slice(lo - p * case["page"], hi - p * case["page"])
                t["k_pages"][at, :, rows] = t["k"][tok].transpose(0, 1)
                t["v_pages"][at, :, rows] = s["v_in"][tok].double().transpose(0, 1)
        return t
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if kind == "prompt":
        first = s["starts"].tolist()
        for i in range(b):
            of = slice(first[i], first[i + 1])
            n = first[i + 1] - first[i]
            hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            for j in range(h):
                x = s["q"][of, j].double() @ s["k"][of, j // g].double().T / math.sqrt(d)
                out[of, j] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ s["v"][of, j // g].double()
        return out
    for i, n in enumerate(s["lens"].tolist()):
        at = s["table"][i, :-(-n // case["page"])].long()
        k, v = (s[x][at].double().transpose(0, 1).reshape(hkv, -1, d)[:, :n] for x in ("k_pages", "v_pages"))
        for j in range(hkv):
            heads = slice(j * g, (j + 1) * g)
            out[i, heads] = torch.softmax(s["q"][i, heads].double() @ k[j].T / math.sqrt(d), -1) @ v[j]
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    kind, b, h, hkv, d = (case[x] for x in ("kind", "batch", "heads", "kv_heads", "dim"))
    lens = _lengths(case)
    if kind == "append":  # q in and out, k in, out and into its page, v in and into its page; the table rows of the positions
        t = sum(lens) if case["prompt"] else b
        positions = case["longest"] if case["prompt"] else len(set(lens))
        return {"bytes": t * d * (4 * h + 10 * hkv) + 4 * d * positions, "flops": t * d * (h + hkv) * (7 if case["norm"] else 3)}
    if kind == "prompt":
        return {"bytes": sum(lens) * d * (4 * h + 4 * hkv), "flops": 4 * h * d * sum(n * (n + 1) // 2 for n in lens)}
    keys = case["shared"] + sum(n - case["shared"] for n in lens)
    return {"bytes": 4 * hkv * d * keys + 4 * b * h * d, "flops": 4 * h * d * sum(lens)}
