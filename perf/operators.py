"""Cases of the row-scaled 8-bit KV cache and of attention under a score rule, each in its plain form and through the library.

Four operators, and what a case of each stands for:

* ``append``  - the KV append (RMSNorm(1+w) of Q and K, RoPE) into a cache whose rows are quantised to 8 bits as they are
  written, one scale per row and kv head; beside the cache it hands out the rotated Q, the gate, and the K/V rows as the
  cache holds them, in 16 bits, for the attention of the same step.
* ``read``    - listed row ranges of such a cache read back as 16-bit rows (the context of a prompt's next chunk, or of a
  prefix that moves to another cache).
* ``decode``  - attention of one new token per sequence over a 16-bit or a row-scaled cache, one allocation or paged, under
  a score rule: scale, tanh cap, distance bias, window, prefix rows, document start.
* ``prefill`` - attention of many tokens per sequence (whole prompts, or a chunk behind rows that are in the cache), packed
  token-major, under the same rule.
"""
import math
import random

import torch

own = False

CODE_MAX = 127.0
SCALE_MIN, SCALE_MAX = 2.0 ** -60, 2.0 ** 60
EPS = 1e-6
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    append = dict(op="append", theta=1e6, interleaved=True, norm=True, gate=False, ragged=False, page_rows=0, type="bf16")
    read = dict(op="read", type="bf16", page_rows=0)
    decode = dict(op="decode", type="bf16", cache="16", page_rows=0, cap=0.0, bias=False, window=0, prefix=0, docs=False, empty=False, lens=1)
    prefill = dict(op="prefill", type="bf16", page_rows=0, cap=0.0, bias=False, window=0, prefix=0, docs=False, pads=False, lens=1)
    return [
        # one token of each of 32 sequences: what every layer does once per generated token, bound by its latency
        dict(append, name="append 32 tokens", hd=128, nkv=8, group=4, seqs=32, tokens=1, rotary=128, first=4000),
        # prompts of the gated-attention layer shape: head_dim 256, a quarter of it rotated, Q and gate side by side
        dict(append, name="append 16k tokens gated", hd=256, nkv=2, group=8, seqs=4, tokens=4096, rotary=64, gate=True, theta=1e7, first=0),
        # the rows of a few short sequences out of small pages, odd lengths and starts
        dict(read, name="read ragged pages", hd=128, nkv=2, seqs=5, rows=700, page_rows=16, type="f16", lens=3),
        # a long shared context back to 16 bits before a chunk of prompts attends to it
        dict(read, name="read 128k rows", hd=128, nkv=8, seqs=4, rows=32768, lens=0),
        # a single short chat turn with capped scores: the smallest call
        dict(decode, name="decode short capped", hd=128, nkv=2, group=8, seqs=1, rows=512, cap=50.0, lens=0),
        # the ragged serving batch (32 sequences of up to 8k rows) on a row-scaled cache, one sequence not started yet
        dict(decode, name="decode ragged row-scaled", hd=128, nkv=8, group=4, seqs=32, rows=8192, cache="rowq", type="f16", cap=30.0, empty=True, lens=2),
        # long sequences of which a window and the first rows are seen, in pages
        dict(decode, name="decode window pages", hd=128, nkv=8, group=5, seqs=48, rows=16384, page_rows=64, window=1023, prefix=4, lens=5),
        # one long context with a distance bias, head_dim 256, row-scaled
        dict(decode, name="decode 128k row-scaled", hd=256, nkv=4, group=4, seqs=1, rows=131072, cache="rowq", bias=True, lens=0),
        # a handful of short prompts of odd lengths, capped scores
        dict(prefill, name="prefill short ragged", hd=128, nkv=2, group=8, seqs=7, tokens=301, context=0, cap=50.0, type="f16", lens=4),
        # the prompt batch of the benchmark with capped scores
        dict(prefill, name="prefill 4x4096 capped", hd=128, nkv=8, group=4, seqs=4, tokens=4096, context=0, cap=50.0, lens=0),
        # documents packed into one long row of tokens, windowed, a few pad tokens that see nothing
        dict(prefill, name="prefill packed documents", hd=128, nkv=8, group=4, seqs=1, tokens=8192, context=0, window=2048, docs=True, pads=True, lens=6),
        # a chunk of a prompt behind rows that are in the cache, in pages, a prefix seen both ways, distance bias
        dict(prefill, name="prefill chunk hd256", hd=256, nkv=2, group=8, seqs=2, tokens=1024, context=8192, page_rows=128, prefix=8500, bias=True, lens=7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "prefill", "prefill"])
    kind = rng.choice(["f16", "bf16"])
    lens = rng.randint(1, 1 << 20)
    if op == "append":
        hd, nkv, group = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
        tokens = _log(rng, 1, 4096)
        most = max(1, (1 << 25) // (hd * nkv * (group + 2) * tokens))
        return dict(op=op, hd=hd, nkv=nkv, group=group, seqs=_log(rng, 1, min(128, most)), tokens=tokens, rotary=rng.choice([0, hd // 4, hd // 2, hd]),
                    theta=rng.choice([1e4, 1e6, 1e7]), interleaved=rng.random() < 0.6, norm=rng.random() < 0.8, gate=rng.random() < 0.4,
                    ragged=tokens > 1 and rng.random() < 0.5, page_rows=rng.choice([0, 16, 64, 256]), first=_log(rng, 1, 16000) - 1, type=kind, lens=lens)
    if op == "read":
        hd, nkv, seqs = rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 4, 8]), _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, min(65536, (1 << 26) // (hd * nkv * seqs))))
        return dict(op=op, hd=hd, nkv=nkv, seqs=seqs, rows=rows, page_rows=rng.choice([0, 0, 16, 48, 256]), type=kind, lens=lens)
    rule = dict(cap=rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), bias=rng.random() < 0.3, window=rng.choice([0, 0, _log(rng, 1, 4096)]),
                prefix=rng.choice([0, 0, _log(rng, 1, 4096)]), docs=rng.random() < 0.3)
    if op == "decode":
        hd, nkv, group, seqs = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8, 12, 16]), _log(rng, 1, 128)
        rows = _log(rng, 1, max(1, min(131072, (1 << 27) // (hd * nkv * seqs))))
        return dict(op=op, hd=hd, nkv=nkv, group=group, seqs=seqs, rows=rows, type=kind, cache=rng.choice(["16", "rowq"]),
                    page_rows=rng.choice([0, 0, 16, 64, 256]), empty=rng.random() < 0.3, lens=lens, **rule)
    hd, nkv, group, seqs = rng.choice([128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8, 16]), _log(rng, 1, 16)
    tokens = _log(rng, 1, 4096)
    context = rng.choice([0, 0, _log(rng, 1, 8192)])
    while seqs > 1 and seqs * tokens * (tokens + context) * nkv * group > 1 << 30:
        seqs -= 1
    while tokens * (tokens + context) * nkv * group > 1 << 30:
        tokens, context = (tokens + 1) // 2, context // 2
    return dict(op=op, hd=hd, nkv=nkv, group=group, seqs=seqs, tokens=tokens, context=context, type=kind, page_rows=rng.choice([0, 0, 16, 32, 128, 256]),
                pads=rng.random() < 0.3, lens=lens, **rule)


def _spread(case, most, least=1):
    """Lengths of the case's sequences: all `most` where lens is 0, else spread by their logarithm, the first one `most`."""
    if not case["lens"] or case["seqs"] == 1 and case["op"] != "read":
        return [most] * case["seqs"]
    r = random.Random(case["lens"])
    return [most] + [_log(r, max(1, min(least, most)), most) for _ in range(case["seqs"] - 1)]


def _append_tokens(case):
    return _spread(case, case["tokens"]) if case["ragged"] else [case["tokens"]] * case["seqs"]


def _append_first(case):
    r = random.Random(case["first"] + 7)
    return [r.randint(0, case["first"]) for _ in range(case["seqs"])]


def _read_ranges(case):
    """(first row, rows) of every sequence."""
    if not case["lens"]:
        return [(0, case["rows"])] * case["seqs"]
    r = random.Random(case["lens"] + 1)
    ends = _spread(case, case["rows"])
    firsts = [r.randint(0, max(0, e // 3)) for e in ends]
    return [(f, e - f) for f, e in zip(firsts, ends)]


def _decode_lens(case):
    lens = _spread(case, case["rows"], max(1, case["rows"] // 16))
    if case["empty"] and len(lens) > 1:
        lens[-1] = 0
    return lens


def _prefill_lens(case):
    """(tokens, rows in the cache before them) of every sequence."""
    tokens = _spread(case, case["tokens"])
    r = random.Random(case["lens"] + 2)
    return [(t, case["context"] if i == 0 or not case["lens"] else r.randint(0, case["context"])) for i, t in enumerate(tokens)]


def _prefixes(case, rows):
    return [min(case["prefix"], n) for n in rows]


def _doc_starts(case):
    """Decode: first visible row of every sequence.  Prefill: of every packed token; -1 for a token that sees no row."""
    r = random.Random(case["lens"] + 3)
    if case["op"] == "decode":
        return [r.randint(0, max(0, n - 1)) // 2 for n in _decode_lens(case)]
    out = []
    for t, c in _prefill_lens(case):
        start = 0
        for i in range(t):
            if case["docs"] and i and r.random() < 1.0 / 500:
                start = c + i
            out.append(start)
        if case["pads"]:
            for i in range(min(t - 1, 3)):
                out[-1 - i] = -1
    return out


def work(case):
    hd, nkv = case["hd"], case["nkv"]
    row8 = nkv * (hd + 4) * 2                                    # codes and scales of one cache row, K and V
    if case["op"] == "append":
        n, nh = sum(_append_tokens(case)), nkv * case["group"]
        q = nh * hd * (1 + case["gate"]) * 2 + 2 * nkv * hd * 2  # in
        o = nh * hd * 2 + (nh * hd * 4 if case["gate"] else 0) + row8 + 2 * nkv * hd * 2
        return {"bytes": n * (q + o), "flops": n * (nh + 2 * nkv) * hd * 8}
    if case["op"] == "read":
        n = sum(c for _, c in _read_ranges(case))
        return {"bytes": n * (row8 + 2 * nkv * hd * 2), "flops": n * nkv * hd * 2}
    nh = nkv * case["group"]
    if case["op"] == "decode":
        lens = _decode_lens(case)
        docs = _doc_starts(case) if case["docs"] else [0] * len(lens)
        pre = _prefixes(case, lens)
        seen = 0
        for n, d, p in zip(lens, docs, pre):
            lo = max(d, n - case["window"]) if case["window"] else d
            seen += max(0, n - lo) + max(0, min(p, lo) - d)
        row = row8 if case["cache"] == "rowq" else nkv * hd * 4
        return {"bytes": seen * row + len(lens) * nh * (hd * 4 + 4), "flops": 4 * seen * nh * hd}
    lens = _prefill_lens(case)
    docs = _doc_starts(case) if case["docs"] or case["pads"] else None
    pre = _prefixes(case, [t + c for t, c in lens])
    pairs = at = 0
    for (t, c), p in zip(lens, pre):
        for i in range(t):
            d = docs[at + i] if docs else 0
            pos = c + i
            if d >= 0:
                lo = max(d, pos + 1 - case["window"]) if case["window"] else d
                pairs += max(0, pos + 1 - lo) + max(0, min(p, lo) - d) + max(0, p - max(pos + 1, d))
        at += t
    n, rows = sum(t for t, _ in lens), sum(t + c for t, c in lens)
    return {"bytes": n * nh * (hd * 4 + 4) + rows * nkv * hd * 4, "flops": 4 * pairs * nh * hd}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def _quantised(x):
    """Codes (stored with 128 added) and scales of rows [..., hd]."""
    scale = (x.abs().amax(-1) / CODE_MAX).clamp(SCALE_MIN, SCALE_MAX)
    code = torch.round(x / scale[..., None]).clamp(-CODE_MAX, CODE_MAX)
    return (code + 128).to(torch.uint8), scale


def _table(case, rows, g):
    """Page table for sequences of the given capacities, pages in random order; (table, pages)."""
    pr = case["page_rows"]
    need = [(n + pr - 1) // pr for n in rows]
    total, width = max(1, sum(need)), max(1, max(need))
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(rows), width, dtype=torch.int32, device="cuda")
    for i, (a, n) in enumerate(zip(_starts(need), need)):
        table[i, :n] = order[a:a + n]
    return table, total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hd, nkv, S, dt = case["hd"], case["nkv"], case["seqs"], TYPES[case["type"]]
    pr = case["page_rows"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    st = {"case": case}

    def pool(rows):
        """Leading dimensions of a cache for sequences of the given capacities."""
        if pr:
            st["table"], pages = _table(case, rows, g)
            return (pages, pr)
        return (len(rows), max(1, max(rows)))

    if case["op"] == "append":
        tokens, first, nh = _append_tokens(case), _append_first(case), nkv * case["group"]
        n = sum(tokens)
        spread = torch.exp(0.5 * randn(n, 1, 1))                 # projections of different tokens differ in size
        st["q"] = (randn(n, nh, hd * (1 + case["gate"])) * spread).to(dt)
        st["k"] = (randn(n, nkv, hd) * spread).to(dt)
        st["v"] = (randn(n, nkv, hd) * spread).to(dt)
        st["w"] = (randn(2, hd) * 0.1).to(torch.bfloat16)
        st["pos"], st["starts"] = _ints(first), _ints(_starts(tokens))
        lead = pool([f + t for f, t in zip(first, tokens)])
        st["codes"] = [torch.zeros(*lead, nkv, hd, dtype=torch.uint8, device="cuda") for _ in range(2)]
        st["scales"] = [torch.zeros(*lead, nkv, device="cuda") for _ in range(2)]
        st["out"] = [torch.empty(n, nh, hd, dtype=dt, device="cuda"), torch.empty(n, nh, hd, device="cuda") if case["gate"] else None,
                     torch.empty(n, nkv, hd, dtype=dt, device="cuda"), torch.empty(n, nkv, hd, dtype=dt, device="cuda")]
        return _ready(st)
    if case["op"] == "read":
        ranges = _read_ranges(case)
        lead = pool([f + n for f, n in ranges])
        st["codes"], st["scales"] = [], []
        for _ in range(2):
            c, s = _quantised(randn(*lead, nkv, hd))
            st["codes"].append(c)
            st["scales"].append(s)
        st["first"], st["starts"] = _ints([f for f, _ in ranges]), _ints(_starts([n for _, n in ranges]))
        n = sum(c for _, c in ranges)
        st["out"] = [torch.empty(n, nkv, hd, dtype=dt, device="cuda") for _ in range(2)]
        return _ready(st)
    nh = nkv * case["group"]
    if case["bias"]:                                             # one slope for each head, falling geometrically
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)], device="cuda")
    if case["op"] == "decode":
        lens = _decode_lens(case)
        lead = pool(lens)
        k, v = randn(*lead, nkv, hd), randn(*lead, nkv, hd)
        if case["cache"] == "rowq":
            st["codes"], st["scales"] = map(list, zip(_quantised(k), _quantised(v)))
        else:
            st["k"], st["v"] = k.to(dt), v.to(dt)
        del k, v
        st["q"], st["lens"] = (2 * randn(S, nh, hd)).to(dt), _ints(lens)
        st["prefix"] = _ints(_prefixes(case, lens)) if case["prefix"] else None
        st["docs"] = _ints(_doc_starts(case)) if case["docs"] else None
        st["out"] = [torch.empty(S, nh, hd, dtype=dt, device="cuda"), torch.empty(S, nh, device="cuda")]
        return _ready(st)
    lens = _prefill_lens(case)
    n, rows = sum(t for t, _ in lens), [t + c for t, c in lens]
    if pr:
        lead = pool(rows)
    else:
        lead = (sum(rows),)
        st["kv_starts"] = _ints(_starts(rows)[:-1])
    st["k"], st["v"] = randn(*lead, nkv, hd).to(dt), randn(*lead, nkv, hd).to(dt)
    st["q"] = (2 * randn(n, nh, hd)).to(dt)
    st["starts"], st["lens"] = _ints(_starts([t for t, _ in lens])), _ints(rows)
    st["prefix"] = _ints(_prefixes(case, rows)) if case["prefix"] else None
    st["docs"] = _ints(_doc_starts(case)) if case["docs"] or case["pads"] else None
    st["out"] = [torch.empty(n, nh, hd, dtype=dt, device="cuda"), torch.empty(n, nh, device="cuda")]
    return _ready(st)


_context = None


def _ready(st):
    """What a program keeps beside its buffers: the context, the views of its caches, the rule and the workspace."""
    if own:
        global _context
        from shady_thinker_b200 import ops
        from shady_thinker_b200.gpu import GpuContext
        case = st["case"]
        if _context is None:
            _context = GpuContext(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream or 1)   # 1: the default stream
        st["gpu"] = _context
        st["code"] = ops.dtype_code(TYPES[case["type"]])
        table = dict(page_table=st.get("table"), page_rows=case["page_rows"], max_pages_per_seq=st["table"].shape[1]) if case["page_rows"] else {}
        if "codes" in st:
            st["view"] = ops.RowqCacheView(st["codes"][0], st["codes"][1], st["scales"][0], st["scales"][1],
                                           seq_rows=0 if table else st["codes"][0].shape[1], **table)
        else:
            st["view"] = ops.KvCacheView(st["code"], st["k"], st["v"], 0 if table or case["op"] == "prefill" else st["k"][0].numel(), **table)
        if case["op"] in ("decode", "prefill"):
            st["rule"] = ops.ScoreRule(cap=case["cap"], slopes=st.get("slopes"), window=case["window"], prefix_lens=st["prefix"], doc_start=st["docs"])
        if case["op"] == "decode":
            shape = dict(head_dim=case["hd"], num_kv_heads=case["nkv"], num_q_heads=case["nkv"] * case["group"], num_seqs=case["seqs"])
            st["ws_bytes"] = ops.decode_rule_workspace_size(_context, **shape)
            st["ws"] = torch.empty(st["ws_bytes"], dtype=torch.uint8, device="cuda")
            ops.decode_rule_workspace_init(_context, st["ws"], st["ws_bytes"], **shape)
    return st


def run(st):
    case = st["case"]
    return (_run_own if own else _run_plain)[case["op"]](case, st)


# ---- through the library --------------------------------------------------------------------------------------------

def _own_append(case, st):
    from shady_thinker_b200 import ops
    q, gate, k, v = st["out"]
    ops.kv_append_rowq(st["gpu"], q_proj_full=st["q"], k_proj=st["k"], v_proj=st["v"], q_out=q, q_gate=gate, k_out=k, v_out=v,
                       cache=st["view"], pos_start=st["pos"], num_heads=case["nkv"] * case["group"], num_kv_heads=case["nkv"],
                       head_dim=case["hd"], rope_theta=case["theta"], rotary_dim=case["rotary"], interleaved=case["interleaved"],
                       eps=EPS, qk_norm_bf16=st["w"] if case["norm"] else None, num_seqs=case["seqs"], tokens_per_seq=case["tokens"],
                       tok_start=st["starts"] if case["ragged"] else None, total_tokens=st["q"].shape[0],
                       in_dtype=st["code"], q_dtype=st["code"], has_gate=case["gate"])
    return {"q": q, "gate": gate, "k": k, "v": v}


def _own_read(case, st):
    from shady_thinker_b200 import ops
    k, v = st["out"]
    ops.kv_read_rowq(st["gpu"], cache=st["view"], k_out=k, v_out=v, row_start=st["first"], out_start=st["starts"], total_rows=k.shape[0],
                     num_seqs=case["seqs"], num_kv_heads=case["nkv"], head_dim=case["hd"], out_dtype=st["code"])
    return {"k": k, "v": v}


def _own_decode(case, st):
    from shady_thinker_b200 import ops
    out, lse = st["out"]
    ops.attn_decode_rule(st["gpu"], q=st["q"], cache=st["view"], seq_lens=st["lens"], out=out, lse=lse, rule=st["rule"], head_dim=case["hd"],
                         num_kv_heads=case["nkv"], num_q_heads=case["nkv"] * case["group"], num_seqs=case["seqs"], q_dtype=st["code"],
                         out_dtype=st["code"], workspace=st["ws"], workspace_bytes=st["ws_bytes"])
    return {"out": out, "lse": lse}


def _own_prefill(case, st):
    from shady_thinker_b200 import ops
    out, lse = st["out"]
    ops.attn_prefill_rule(st["gpu"], q=st["q"], cache=st["view"], q_starts=st["starts"], kv_starts=st.get("kv_starts"), kv_lens=st["lens"],
                          out=out, lse=lse, rule=st["rule"], head_dim=case["hd"], num_kv_heads=case["nkv"],
                          num_q_heads=case["nkv"] * case["group"], num_seqs=case["seqs"], total_q=st["q"].shape[0],
                          cache_rows=st["k"].numel() // (case["nkv"] * case["hd"]), dtype=st["code"])
    return {"out": out, "lse": lse}


_run_own = {"append": _own_append, "read": _own_read, "decode": _own_decode, "prefill": _own_prefill}


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _token_rows(starts, first, n):
    """Sequence and cache row of each of n packed tokens."""
    at = torch.arange(n, device="cuda")
    seq = torch.searchsorted(starts[1:].long(), at, right=True)
    return seq, first.long()[seq] + at - starts.long()[seq]


def _cache_index(case, st, seq, row):
    """The two leading indices of a cache row of a sequence."""
    if case["page_rows"]:
        return st["table"].long()[seq, row // case["page_rows"]], row % case["page_rows"]
    return seq, row


def _rotated(x, case, pos):
    """RoPE of the first `rotary` dims of x [n, heads, hd] at positions pos [n]; angles in 64 bits."""
    rd = case["rotary"]
    if not rd:
        return x
    freq = case["theta"] ** (-torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    r, rest = x[..., :rd], x[..., rd:]
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :rd // 2], r[..., rd // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1)


def _plain_append(case, st):
    hd, n, dt = case["hd"], st["q"].shape[0], TYPES[case["type"]]
    seq, pos = _token_rows(st["starts"], st["pos"], n)
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    gate = q[..., hd:] if case["gate"] else None
    q = q[..., :hd]
    if case["norm"]:
        w = 1 + st["w"].float()
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * w[0]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * w[1]
    q, k = _rotated(q, case, pos), _rotated(k, case, pos)
    held = []
    for x, codes, scales in zip((k, v), st["codes"], st["scales"]):
        c, s = _quantised(x)
        at = _cache_index(case, st, seq, pos)
        codes[at], scales[at] = c, s
        held.append(((c.float() - 128) * s[..., None]).to(dt))
    return {"q": q.to(dt), "gate": gate.contiguous() if gate is not None else None, "k": held[0], "v": held[1]}


def _plain_read(case, st):
    seq, row = _token_rows(st["starts"], st["first"], st["out"][0].shape[0])
    at = _cache_index(case, st, seq, row)
    k, v = (((c[at].float() - 128) * s[at][..., None]).to(TYPES[case["type"]]) for c, s in zip(st["codes"], st["scales"]))
    return {"k": k, "v": v}


def _rows(case, st):
    """K and V in 32 bits as [seqs, rows, nkv, hd], rows behind a sequence's end among them."""
    if "codes" in st:
        kv = [(c.float() - 128) * s[..., None] for c, s in zip(st["codes"], st["scales"])]
    else:
        kv = [st["k"], st["v"]]
    if case["page_rows"]:
        return [x[st["table"].long()].flatten(1, 2).float() for x in kv]
    if "kv_starts" in st:
        most = int(max(t + c for t, c in _prefill_lens(case)))
        at = (st["kv_starts"].long()[:, None] + torch.arange(most, device="cuda")).clamp_(max=kv[0].shape[0] - 1)
        return [x[at].float() for x in kv]
    return [x.float() for x in kv]


def _attend(case, st, q, pos, n_rows, docs):
    """q [S, T, nh, hd] at positions pos [S, T] over the first n_rows [S] cache rows; docs [S, T] first visible row or None."""
    hd, nkv, G = case["hd"], case["nkv"], case["group"]
    S, T = pos.shape
    k, v = _rows(case, st)
    R = k.shape[1]
    q = q.float().view(S, T, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, G * T, hd)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).view(S, nkv, G, T, R)
    del k
    s *= 1 / math.sqrt(hd)
    if case["cap"]:
        s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
    row = torch.arange(R, device="cuda")
    away = pos[:, :, None] - row                                 # [S, T, R]
    if case["bias"]:
        s -= st["slopes"].view(nkv, G, 1, 1) * away[:, None, None].abs().float()
    seen = away >= 0
    if case["window"]:
        seen &= away < case["window"]
    if case["prefix"]:
        seen |= row < st["prefix"].long()[:, None, None]
    if docs is not None:
        seen &= row >= docs[:, :, None]
    seen &= row < n_rows[:, None, None]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((row < n_rows[:, None])[..., None, None], v, torch.zeros_like(v))
    o = torch.matmul(p.view(S, nkv, G * T, R), v.transpose(1, 2)).view(S, nkv, G, T, hd)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    lse = (m + total.log())[..., 0]
    return o.permute(0, 3, 1, 2, 4).reshape(S, T, nkv * G, hd).to(TYPES[case["type"]]), lse.permute(0, 3, 1, 2).reshape(S, T, nkv * G)


def _plain_decode(case, st):
    n = st["lens"].long()
    docs = st["docs"].long()[:, None] if case["docs"] else None
    out, lse = _attend(case, st, st["q"][:, None], n[:, None] - 1, n, docs)
    return {"out": out[:, 0], "lse": lse[:, 0]}


def _plain_prefill(case, st):
    lens = _prefill_lens(case)
    n, T = st["q"].shape[0], max(t for t, _ in lens)
    seq, at = _token_rows(st["starts"], torch.zeros_like(st["lens"]), n)
    q = st["q"].new_zeros(case["seqs"], T, *st["q"].shape[1:])
    q[seq, at] = st["q"]
    tokens = st["starts"][1:].long() - st["starts"][:-1].long()
    pos = (st["lens"].long() - tokens)[:, None] + torch.arange(T, device="cuda")
    docs = None
    if st["docs"] is not None:
        d = st["docs"].long()
        docs = torch.zeros(case["seqs"], T, dtype=torch.long, device="cuda")
        docs[seq, at] = torch.where(d < 0, 1 << 32, d)
    out, lse = _attend(case, st, q, pos, st["lens"].long(), docs)
    return {"out": out[seq, at], "lse": lse[seq, at]}


_run_plain = {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "prefill": _plain_prefill}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------

def _held64(x):
    """What a row-scaled cache holds of rows x [..., hd]: scale = largest magnitude / 127, codes to the nearest."""
    top = x.abs().max(-1, keepdim=True).values
    step = (top / 127).clamp(2.0 ** -60, 2.0 ** 60)
    return torch.clamp(torch.round(x / step), -127, 127) * step


def _norm_rope64(x, w, case, pos):
    x = x.double()
    if case["norm"]:
        x = x / ((x * x).sum(-1, keepdim=True) / case["hd"] + EPS).sqrt() * (1 + w.double())
    y = x.clone()
    half = case["rotary"] // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        t = pos.double() / case["theta"] ** (2 * i / case["rotary"])
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def _exact_rows(case, st, s, n):
    """The first n rows of sequence s, K and V as [n, nkv, hd] in 64 bits."""
    rows = torch.arange(n, device="cuda")
    if case["page_rows"]:
        at = (st["table"][s].long()[rows // case["page_rows"]], rows % case["page_rows"])
    elif "kv_starts" in st:
        at = (int(st["kv_starts"][s]) + rows,)
    else:
        at = (torch.full_like(rows, s), rows)
    if "codes" in st:
        return [(c[at].double() - 128.0) * f[at].double().unsqueeze(-1) for c, f in zip(st["codes"], st["scales"])]
    return [st["k"][at].double(), st["v"][at].double()]


def _exact_attention(case, st, s, h, q, pos, k, v, docs):
    """One head: q [T, hd] at positions pos [T] over k, v [n, hd]."""
    z = q.double() @ k.T / math.sqrt(case["hd"])
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    j, i = torch.arange(k.shape[0], device="cuda")[None, :], pos[:, None]
    if case["bias"]:
        z = z - float(st["slopes"][h]) * (i - j).abs().double()
    near = (j <= i) & ((i - j < case["window"]) if case["window"] else (j >= 0))
    if st["prefix"] is not None:
        near = near | (j < int(st["prefix"][s]))
    if docs is not None:
        near = near & (j >= docs[:, None])
    z = torch.where(near, z, torch.full_like(z, -math.inf))
    lse = torch.logsumexp(z, -1)
    p = torch.where(near, torch.exp(z - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(z))
    return p @ v, lse


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    hd, nkv, G = case["hd"], case["nkv"], case["group"] if "group" in case else 1
    if case["op"] == "append":
        tokens, first = _append_tokens(case), _append_first(case)
        pos = torch.cat([torch.arange(f, f + t, device="cuda") for f, t in zip(first, tokens)])
        return {"q": _norm_rope64(st["q"][..., :hd], st["w"][0], case, pos), "gate": st["q"][..., hd:].double() if case["gate"] else None,
                "k": _held64(_norm_rope64(st["k"], st["w"][1], case, pos)), "v": _held64(st["v"].double())}
    if case["op"] == "read":
        got = [_exact_rows(case, st, s, f + n) for s, (f, n) in enumerate(_read_ranges(case))]
        return {n: torch.cat([g[i][f:] for g, (f, _) in zip(got, _read_ranges(case))]) for i, n in enumerate("kv")}
    nh = nkv * G
    if case["op"] == "decode":
        out, lse = torch.zeros(case["seqs"], nh, hd, dtype=torch.float64, device="cuda"), torch.full((case["seqs"], nh), -math.inf, dtype=torch.float64, device="cuda")
        docs = _doc_starts(case) if case["docs"] else None
        for s, n in enumerate(_decode_lens(case)):
            if n:
                k, v = _exact_rows(case, st, s, n)
                at = torch.tensor([n - 1], device="cuda")
                d = torch.tensor([docs[s]], device="cuda") if docs else None
                for h in range(nh):
                    o, z = _exact_attention(case, st, s, h, st["q"][s, h][None], at, k[:, h // G], v[:, h // G], d)
                    out[s, h], lse[s, h] = o[0], z[0]
        return {"out": out, "lse": lse}
    n = st["q"].shape[0]
    out, lse = torch.zeros(n, nh, hd, dtype=torch.float64, device="cuda"), torch.zeros(n, nh, dtype=torch.float64, device="cuda")
    docs = [d if d >= 0 else 1 << 32 for d in _doc_starts(case)] if case["docs"] or case["pads"] else None
    a = 0
    for s, (t, c) in enumerate(_prefill_lens(case)):
        k, v = _exact_rows(case, st, s, t + c)
        at = torch.arange(c, c + t, device="cuda")
        d = torch.tensor(docs[a:a + t], device="cuda") if docs else None
        for h in range(nh):
            out[a:a + t, h], lse[a:a + t, h] = _exact_attention(case, st, s, h, st["q"][a:a + t, h], at, k[:, h // G], v[:, h // G], d)
        a += t
    return {"out": out, "lse": lse}
