"""The 4-bit key/value cache: writing it, reading it back, and attention over it, as a serving program uses them.

A cache holds signed 4-bit codes in pages, ``k_codes`` and ``v_codes`` uint8 [pages, kv_heads, page_size, head_dim / 2] (the
low nibble is the even channel, two's complement), and one bfloat16 scale for each token, head and group of ``group`` channels,
``scales`` [pages, kv_heads, page_size, 2, head_dim / group] (0: keys, 1: values). Token t of sequence b is row t % page_size
of page ``block_table[b, t // page_size]``. ``cu_q`` says which rows of a packed [rows, heads, head_dim] tensor belong to a
sequence: they are its last ones, at positions seq_len - n .. seq_len - 1.

  writing:  a = max |x| of a group, s = the smallest bfloat16 not below a / 7, code = x / s rounded to the nearest, ties to even
  reading:  code * s
  attention of the query at position p over 0 <= t <= p (or t < seq_len, not causal) and t > p - window (window > 0):
            softmax(q . k_t / sqrt(head_dim)) . v_t
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _case(name, op, dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim, group, page, ragged=False, causal=True,
          window=0):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "q_len": q_len, "kv_len": kv_len, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "group": group, "page": page, "ragged": ragged, "causal": causal,
            "window": window}


def listed():
    return [
        # One token of one sequence enters the cache: a chat's decode step, where a launch is all there is.
        _case("write_decode_1", "write", "fp16", 1, 1, 700, 8, 8, 128, 64, 16),
        # The decode step of a full batch: one token of each sequence, each to a page of its own.
        _case("write_decode_64", "write", "bf16", 64, 1, 1500, 8, 8, 128, 32, 16, ragged=True),
        # Prompts of several lengths enter at once, in float32 (the linear layers' own type), 96 channels a head.
        _case("write_prompts_fp32", "write", "fp32", 5, 1237, 1237, 12, 12, 96, 32, 48, ragged=True),
        # A large chunk of prompts: 16 k tokens of 8 heads.
        _case("write_chunk_16k", "write", "bf16", 4, 4096, 4096, 8, 8, 128, 64, 64),
        # A short prefix is read back, to be joined to a cache of another kind.
        _case("read_prefix", "read", "fp16", 1, 77, 77, 4, 4, 64, 64, 16),
        # A whole cache is read back: long sequences handed over to another program.
        _case("read_long", "read", "bf16", 4, 16384, 16384, 8, 8, 128, 64, 64),
        # Decode of one short chat: latency.
        _case("attend_decode_short", "attend", "fp16", 1, 1, 129, 16, 4, 64, 32, 16),
        # Decode of one very long document: the cache is split over the whole GPU.
        _case("attend_decode_128k", "attend", "bf16", 1, 1, 131072, 32, 8, 128, 64, 256),
        # Decode of a full batch of uneven lengths: the serving loop.
        _case("attend_decode_64", "attend", "bf16", 64, 1, 8192, 64, 8, 128, 32, 64, ragged=True),
        # Speculative decoding in float32, five tokens a sequence, one head a key head, odd pages and lengths.
        _case("attend_draft_fp32", "attend", "fp32", 7, 5, 2011, 12, 12, 96, 32, 48, ragged=True),
        # Chunked prefill of uneven prompts over what is cached, within a sliding window.
        _case("attend_chunk_window", "attend", "fp16", 6, 700, 3500, 16, 4, 64, 64, 32, ragged=True, window=1024),
        # A long prompt's prefill over its own cache: bound by the matrix products.
        _case("attend_prefill_8k", "attend", "bf16", 1, 8192, 8192, 32, 8, 128, 64, 64),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    top = {}
    for c in listed():
        w = work(c)
        top[c["op"]] = max(top.get(c["op"], 0), max(w["bytes"], _cost(c)))
    while True:
        op = rng.choice(("write", "read", "attend", "attend", "attend"))
        head_dim = rng.choice((64, 96, 128, 128, 192, 256))
        group = rng.choice([g for g in (32, 64, 128) if head_dim % g == 0])
        kv_heads = rng.choice((1, 2, 3, 4, 8, 16))
        batch, kv_len = log(1, 64), log(1, 65536)
        if op == "attend":
            q_len = 1 if rng.random() < 0.5 else log(2, 4096)
        else:
            q_len = log(1, 16384)
        q_len = min(q_len, kv_len)
        c = _case("", op, rng.choice(("fp16", "bf16", "fp32")), batch, q_len, kv_len,
                  kv_heads * (rng.choice((1, 2, 4, 5, 8, 12)) if op == "attend" else 1), kv_heads, head_dim, group,
                  rng.choice((16, 16, 32, 48, 64, 100, 256)), rng.random() < 0.6, rng.random() < 0.8,
                  log(16, 8192) if rng.random() < 0.25 else 0)
        del c["name"]
        if op != "attend":
            c["causal"], c["window"] = True, 0
        if max(work(c)["bytes"], _cost(c)) <= top[op]:
            return c


def _cost(c):
    """What the plain form of a case moves, so that a drawn one does not cost more than the listed ones."""
    lens, _ = _lengths(c)
    rows = len(lens) * max(lens) * c["kv_heads"] * c["head_dim"] * 8
    pairs = len(lens) * c["q_len"] * max(lens) * c["q_heads"] * 8 if c["op"] == "attend" else 0
    return float(rows + pairs)


def _lengths(c):
    """Lengths of the sequences and how many rows of each come with the call."""
    b, full = c["batch"], c["kv_len"]
    lens = [max(1, full * (1 + (5 * i) % b) // b) if c["ragged"] else full for i in range(b)]
    return lens, [min(n, max(1, c["q_len"] - (13 * i) % max(1, c["q_len"] // 2)) if c["ragged"] else c["q_len"])
                  for i, n in enumerate(lens)]


def _visible(c, n, q):
    """Tokens that some query of one sequence sees, and the number of pairs of query and token."""
    pairs, low = 0, n
    for i in range(q):
        p = n - q + i
        end = p + 1 if c["causal"] else n
        start = min(end, max(0, p - c["window"] + 1)) if c["window"] else 0
        pairs += end - start
        low = min(low, start)
    return n - low, pairs


def work(c):
    lens, news = _lengths(c)
    rows, d, h = sum(news), c["head_dim"], c["kv_heads"]
    row = d // 2 + 2 * (d // c["group"])  # bytes of a token and head, of keys or of values
    e = SIZES[c["dtype"]]
    if c["op"] == "write":  # rows in, cache out, and the values that it stands for
        return {"bytes": 2 * rows * h * (2 * d * e + row), "flops": 2 * rows * h * d * 4}
    if c["op"] == "read":
        return {"bytes": 2 * rows * h * (d * e + row), "flops": 2 * rows * h * d}
    seen, pairs = map(sum, zip(*(_visible(c, n, q) for n, q in zip(lens, news))))
    return {"bytes": 2 * seen * h * row + 2 * rows * c["q_heads"] * d * e, "flops": 4 * d * pairs * c["q_heads"]}


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, d, page, dt = c["kv_heads"], c["head_dim"], c["page"], DTYPES[c["dtype"]]
    lens, news = _lengths(c)
    rows, most = sum(news), -(-max(lens) // page)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3  # a pool with pages of nobody
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.zeros((len(lens), most), dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = torch.arange(at, at + k, dtype=torch.int32)
        at += k
    s = {"case": dict(c), "rows": rows, "max_q": max(news), "max_len": max(lens)}
    s["block_table"] = order[table.long().cuda()].to(torch.int32)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    s["cu_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda")

    # Channels of a model's keys and values differ in size; a few are far larger than the rest.
    size = torch.exp(0.4 * torch.randn((2, h, d), generator=g, device="cuda"))

    def rows_of(n, which):
        return torch.randn((n, h, d), generator=g, device="cuda") * size[which]

    s["scales"] = torch.empty((pages, h, page, 2, d // c["group"]), dtype=torch.bfloat16, device="cuda")
    for which, name in enumerate(("k_codes", "v_codes")):
        s[name] = torch.empty((pages, h, page, d // 2), dtype=torch.uint8, device="cuda")
        piece = max(1, (1 << 26) // (page * h * d))
        for p in range(0, pages, piece):
            m = min(piece, pages - p)
            x = rows_of(m * page, which).view(m, page, h, d).transpose(1, 2).reshape(m, h, page, d // c["group"], c["group"])
            scale = (x.abs().amax(-1) / 7).bfloat16()
            code = (x / scale.float()[..., None]).round().clamp(-7, 7).to(torch.int8).view(m, h, page, d // 2, 2)
            s[name][p:p + m] = ((code[..., 0] & 15) | ((code[..., 1] & 15) << 4)).view(torch.uint8)
            s["scales"][p:p + m, :, :, which] = scale
    if c["op"] == "write":
        s["k"], s["v"] = (rows_of(rows, which).to(dt) for which in (0, 1))
    if c["op"] == "attend":
        s["q"] = torch.randn((rows, c["q_heads"], d), generator=g, device="cuda").to(dt)
    return s


# ---- the plain forms -------------------------------------------------------
def _places(s):
    """Sequence, position, page and row in the page of each packed row."""
    cu, lens, page = s["cu_q"].long(), s["seq_lens"].long(), s["case"]["page"]
    row = torch.arange(s["rows"], device=cu.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = lens[seq] - (cu[seq + 1] - row)
    return seq, pos, s["block_table"].long()[seq, pos // page], pos % page


def _unpack(codes, scales, group):
    """Packed rows [..., d / 2] and their scales [..., d / group] as float32 [..., d]."""
    p = codes.to(torch.int32)
    n = torch.stack((p & 15, p >> 4), dim=-1).flatten(-2)
    n = (n ^ 8) - 8
    return (n.unflatten(-1, (-1, group)).float() * scales.float()[..., None]).flatten(-2)


def _quantise(x, group):
    """x float [n, h, d] -> codes int32 [n, h, d], scales bfloat16 [n, h, d / group]. In 64 bits: the scale is the next bfloat16
    above a quotient, and codes next to a half fall to either side."""
    x = x.double().unflatten(-1, (-1, group))
    a = x.abs().amax(-1)
    s = (a / 7).float().bfloat16()
    up = (s.view(torch.int16) + 1).view(torch.bfloat16)
    s = torch.where(s.double() * 7 < a, up, s)
    code = torch.where(s[..., None] > 0, x / s.double()[..., None], 0.0).round()
    return code.to(torch.int32).flatten(-2), s


def _plain_read(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    _, _, page, at = _places(s)
    return [_unpack(s[n][page, :, at], s["scales"][page, :, at, which], c["group"]).to(dt)
            for which, n in enumerate(("k_codes", "v_codes"))]


def _plain_write(s):
    _, _, page, at = _places(s)
    for which, (x, n) in enumerate((("k", "k_codes"), ("v", "v_codes"))):
        code, scale = _quantise(s[x], s["case"]["group"])
        code = code.unflatten(-1, (-1, 2)) & 15
        s[n][page, :, at] = (code[..., 0] | (code[..., 1] << 4)).to(torch.uint8)
        s["scales"][page, :, at, which] = scale
    return _plain_read(s)


def _plain_attend(s):
    c = s["case"]
    b, h, d, top = c["batch"], c["kv_heads"], c["head_dim"], s["max_len"]
    g, page, lens = c["q_heads"] // h, c["page"], s["seq_lens"].long()
    t = torch.arange(top, device="cuda")
    where = s["block_table"].long()[:, t // page], t % page
    k, v = (_unpack(s[n][where[0], :, where[1]], s["scales"][where[0], :, where[1], which], c["group"]).transpose(1, 2)
            for which, n in enumerate(("k_codes", "v_codes")))  # [b, h, t, d]
    seq, pos, _, _ = _places(s)
    at = pos - (lens - s["cu_q"].long().diff())[seq]  # row among its sequence's own
    q = torch.zeros((b, s["max_q"], h, g, d), device="cuda")
    q[seq, at] = s["q"].float().view(-1, h, g, d)
    scores = q.permute(0, 2, 3, 1, 4).reshape(b, h, -1, d) @ k.transpose(-1, -2)
    scores = scores.view(b, h, g, s["max_q"], top).mul_(1 / math.sqrt(d))
    p = (lens - s["cu_q"].long().diff())[:, None] + torch.arange(s["max_q"], device="cuda")  # [b, q]
    hidden = (t >= lens[:, None, None]) | (p >= lens[:, None])[..., None]
    if c["causal"]:
        hidden = hidden | (t > p[..., None])
    if c["window"]:
        hidden = hidden | (t <= p[..., None] - c["window"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = scores.sum(-1, keepdim=True)
    o = scores.view(b, h, -1, top) @ v / torch.where(total == 0, 1.0, total).view(b, h, -1, 1)
    o = o.view(b, h, g, s["max_q"], d).permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], h * g, d)
    return [o[seq, at].to(DTYPES[c["dtype"]])]


# ---- the framework's calls -------------------------------------------------
def _ext():
    here = str(Path(__file__).resolve().parents[1] / "lsq-lowbit-optimization_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import int4_int8_ext
    return int4_int8_ext


def run(s):
    c = s["case"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[c["op"]](s)
    ext = _ext()
    cache = s["k_codes"], s["v_codes"], s["scales"], s["block_table"], s["seq_lens"]
    if c["op"] == "write":
        ext.kv_cache_write_int4(s["k"], s["v"], *cache, cu_q=s["cu_q"])
    if c["op"] in ("write", "read"):
        return list(ext.kv_cache_read_int4(*cache, rows=s["rows"], dtype=DTYPES[c["dtype"]], cu_q=s["cu_q"]))
    return [ext.attention_int4_kv(s["q"], *cache, cu_q=s["cu_q"], max_q=s["max_q"], max_len=s["max_len"],
                                  causal=c["causal"], window=c["window"])]


# ---- the definition, in 64 bits --------------------------------------------
def _exact_values(codes, scales, group):
    low, high = codes & 0x0F, codes >> 4
    n = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=codes.device)
    n[..., 0::2], n[..., 1::2] = low.double(), high.double()
    n[n > 7] -= 16
    return n * scales.double().repeat_interleave(group, dim=-1)


def _exact_rounded(x, group):
    """What a written row reads back as: x to the nearest multiple of its group's scale."""
    x = x.double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], group):
        part = x[..., at:at + group]
        low = part.abs().max(-1).values / 7
        e = torch.floor(torch.log2(low.clamp_min(1e-30))) - 7  # a bfloat16 holds 8 bits
        step = torch.ceil(low * torch.exp2(-e)) * torch.exp2(e)
        out[..., at:at + group] = torch.round(part / step[..., None]) * step[..., None]
    return out


def exact(c, seed):
    s = prepare(c, seed)
    lens, news = _lengths(c)
    dt, page, group = DTYPES[c["dtype"]], c["page"], c["group"]
    if c["op"] == "write":
        return [_exact_rounded(s[x], group) for x in ("k", "v")]
    outs = [[], []]
    first = 0
    for b, (n, new) in enumerate(zip(lens, news)):
        at = s["block_table"][b, :-(-n // page)].long()
        kv = []
        for which, name in enumerate(("k_codes", "v_codes")):
            codes = s[name][at].transpose(1, 2).flatten(0, 1)[:n]  # [n, h, d / 2]
            scales = s["scales"][at][:, :, :, which].transpose(1, 2).flatten(0, 1)[:n]
            kv.append((codes, scales))
        if c["op"] == "read":
            for o, (codes, scales) in zip(outs, kv):
                o.append(_exact_values(codes[n - new:], scales[n - new:], group))
            continue
        q = s["q"][first:first + new].double()
        first += new
        ratio = c["q_heads"] // c["kv_heads"]
        o = torch.empty_like(q)
        pos = torch.arange(n - new, n, device="cuda")[:, None]
        for h in range(c["kv_heads"]):
            k, v = (_exact_values(codes[:, h], scales[:, h], group) for codes, scales in kv)
            for i in range(0, new, 2048):
                part = slice(i, min(new, i + 2048))
                x = torch.einsum("igd,td->git", q[part, h * ratio:(h + 1) * ratio], k) / math.sqrt(c["head_dim"])
                t = torch.arange(n, device="cuda")
                if c["causal"]:
                    x[:, t > pos[part]] = -math.inf
                if c["window"]:
                    x[:, t <= pos[part] - c["window"]] = -math.inf
                o[part, h * ratio:(h + 1) * ratio] = torch.einsum("git,td->igd", torch.softmax(x, dim=-1), v)
        outs[0].append(o)
    return [torch.cat(o) for o in outs if o]
