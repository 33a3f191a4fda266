"""Operators of a text model beside the image model, as cases that can be timed
and checked: what a prompt's encoder or writer runs on this library's text side
(grouped-query heads of 128, 32 over 8 in the text tower that feeds the DiT).

  rotary     qw_gpu_rotary_bf16: per-head RMS norm and rotary positions of q and
             k, with k and v going into a paged cache or beside q
  attention  qw_gpu_paged_attention_bf16: the new tokens of several sequences
             against all that a paged cache holds of each
  linear     qw_gpu_linear_int4: 4-bit weights with a scale per group of inputs

`own` false computes them in plain torch operations, in 32 bits (angles in 64),
rounded once at the end; true calls the library.
"""
import math

import numpy as np
import torch

own = False

D = 128  # head dimension
EPS = 1e-6
NO_PAGE = -1  # a table entry without a page (0xffffffff)


def listed():
    return [
        # one user's next token: q, k of one row rotated, k and v appended
        dict(name="rotary_step_1", kind="rotary", heads=32, kv_heads=8, sequences=1, new=1,
             past=2048, pad=0, page=64, layout="half", rotary=128, scaling="plain", norm=True,
             cache=True),
        # a prompt far into a long document: half of each head rotated in
        # interleaved pairs, frequencies stretched, no cache
        dict(name="rotary_far_1000", kind="rotary", heads=32, kv_heads=8, sequences=1, new=1000,
             past=400000, pad=0, page=64, layout="interleaved", rotary=64, scaling="yarn",
             norm=False, cache=False),
        # prompts of four users in one call, appended
        dict(name="rotary_prompts_8192", kind="rotary", heads=32, kv_heads=8, sequences=4,
             new=2400, past=300, pad=0, page=64, layout="half", rotary=128, scaling="plain",
             norm=True, cache=True),
        # one user's next token against a short conversation: latency
        dict(name="attention_step_1", kind="attention", heads=32, kv_heads=8, sequences=1, new=1,
             past=2048, pad=0, page=64, window=0, holes=False),
        # a batch of users' next tokens, ragged conversations, small pages
        dict(name="attention_step_64", kind="attention", heads=32, kv_heads=8, sequences=64,
             new=1, past=8191, pad=0, page=16, window=0, holes=False),
        # two users deep into long documents
        dict(name="attention_step_long", kind="attention", heads=32, kv_heads=8, sequences=2,
             new=1, past=131000, pad=0, page=64, window=0, holes=False),
        # a chunk of a long prompt against the chunks before it
        dict(name="attention_chunk_512", kind="attention", heads=32, kv_heads=8, sequences=1,
             new=512, past=7937, pad=0, page=64, window=0, holes=False),
        # fresh prompts of four users, ragged, in one call
        dict(name="attention_prompts", kind="attention", heads=32, kv_heads=8, sequences=4,
             new=4096, past=130, pad=24, page=64, window=0, holes=False),
        # next token of one user: the gate and up projections, the down projection
        dict(name="linear_up_1", kind="linear", rows=1, k=4096, cols=24576, group=128,
             zeros=False, bias=False),
        dict(name="linear_down_1", kind="linear", rows=1, k=12288, cols=4096, group=64,
             zeros=True, bias=False),
        # a batch of users' next tokens through the q|k|v projection
        dict(name="linear_qkv_16", kind="linear", rows=16, k=4096, cols=6144, group=128,
             zeros=False, bias=True),
        # a larger batch, or a short prompt
        dict(name="linear_up_60", kind="linear", rows=60, k=4096, cols=24576, group=128,
             zeros=False, bias=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8), (32, 8), (24, 24), (32, 32), (16, 2), (8, 1), (28, 4), (40, 8)]


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "linear"])
    heads, kv = rng.choice(HEADS)
    page = rng.choice([8, 16, 32, 64, 128, 256])
    if kind == "rotary":
        case = dict(kind=kind, heads=heads, kv_heads=kv, sequences=_log_int(rng, 1, 64),
                    new=_log_int(rng, 1, 4096), past=_log_int(rng, 1, 30000),
                    pad=rng.choice([0, 0, rng.randint(1, 40)]), page=page,
                    layout=rng.choice(["half", "interleaved"]),
                    rotary=rng.choice([128, 128, 64, 96, 32, 24]),
                    scaling=rng.choice(["plain", "linear", "ntk", "parts", "yarn"]),
                    norm=rng.random() < 0.5, cache=rng.random() < 0.6)
        while case["sequences"] > 1 and (case["sequences"] * (case["new"] + case["past"]) > 60000 or
                                         case["sequences"] * case["new"] > 8192):
            case["sequences"] //= 2
    elif kind == "attention":
        case = dict(kind=kind, heads=heads, kv_heads=kv, sequences=_log_int(rng, 1, 64),
                    new=rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)]),
                    past=_log_int(rng, 1, 30000), pad=rng.choice([0, 0, rng.randint(1, 40)]),
                    page=page, window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]),
                    holes=rng.random() < 0.2)
        while case["sequences"] > 1 and (
                case["sequences"] * (case["new"] + case["past"]) * kv > 2000000 or
                case["sequences"] * case["new"] * heads * (case["new"] + case["past"]) > 1 << 29):
            case["sequences"] //= 2
        case["past"] = max(1, min(case["past"], (1 << 29) // (case["sequences"] * case["new"] * heads) -
                               case["new"]))
    else:
        group = rng.choice([32, 64, 128, 128])
        k = group * _log_int(rng, 512 // group, 12288 // group)
        case = dict(kind=kind, rows=_log_int(rng, 1, 64), k=k,
                    cols=8 * _log_int(rng, 16, 24576 * 4096 // k // 8), group=group,
                    zeros=rng.random() < 0.4, bias=rng.random() < 0.4)
    return case


# ---- sizes of a batch: the case alone says them ---------------------------


def _new(case):
    """New tokens of each sequence, ragged between half and all of `new`."""
    n = case["new"]
    return [n - (i * 7919) % (n // 2 + 1) for i in range(case["sequences"])]


def _past(case):
    """Tokens that each sequence holds already."""
    n = case["past"]
    return [n - (i * 104729) % (n // 2 + 1) for i in range(case["sequences"])]


def _rows(case):
    return sum(_new(case)) + case["pad"]


class _State:
    """The inputs and outputs of a case, by attribute."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _bf16(gen, *shape, std=1.0, mean=0.0):
    t = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    flat, step = t.view(-1), 1 << 27
    for i in range(0, flat.numel(), step):
        m = min(step, flat.numel() - i)
        flat[i:i + m] = torch.randn(m, generator=gen, device="cuda") * std + mean
    return t


def _i32(values):
    return torch.tensor(np.asarray(values, dtype=np.int64).astype(np.uint32).view(np.int32),
                        device="cuda")


def _cache(s, case, gen, seed):
    """A paged cache: pages dealt to the sequences in a shuffled order, some
    spare, the table's unused entries without a page."""
    page, lengths = case["page"], [a + b for a, b in zip(_past(case), _new(case))]
    used = [-(-n // page) for n in lengths]
    s.pages, s.table_ld = sum(used) + 3, max(used) + 1
    order = np.random.RandomState(seed % (1 << 31)).permutation(s.pages)
    table = np.full((len(lengths), s.table_ld), NO_PAGE, np.int64)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
        if case.get("holes") and n > 4:  # pages given up from the middle
            table[i, 1 + n // 3] = NO_PAGE
    s.table, s.lengths = _i32(table), _i32(lengths)
    s.starts = _i32(np.concatenate([[0], np.cumsum(_new(case))]))
    s.cache_k = _bf16(gen, s.pages, page, case["kv_heads"], D)
    s.cache_v = _bf16(gen, s.pages, page, case["kv_heads"], D)
    s.longest, s.most = max(lengths), max(_new(case))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = _State(case=dict(case), kept=None)
    if case["kind"] == "linear":
        n, k, cols, group = case["rows"], case["k"], case["cols"], case["group"]
        s.x = _bf16(gen, n, k)
        q = (_bf16(gen, cols, k, std=2.7, mean=7.5).round_().clamp_(0, 15)).to(torch.uint8)
        s.weight = q[:, 0::2] | (q[:, 1::2] << 4)  # input 2 i in the low half of byte i
        s.scales = (torch.rand(cols, k // group, generator=gen, device="cuda") * 0.01 +
                    0.003).to(torch.bfloat16)
        s.zeros = torch.randint(5, 11, (cols, k // group), generator=gen,
                                device="cuda").to(torch.bfloat16) if case["zeros"] else None
        s.bias = _bf16(gen, cols, std=0.1) if case["bias"] else None
        s.out = torch.empty(n, cols, dtype=torch.bfloat16, device="cuda")
    else:
        heads, kv, rows = case["heads"], case["kv_heads"], _rows(case)
        if case["kind"] == "attention":
            s.q = _bf16(gen, rows, heads, D, std=1.5)
            _cache(s, case, gen, seed)
        else:
            s.qkv = _bf16(gen, rows, heads + 2 * kv, D)  # the fused projection's output
            s.norm_q, s.norm_k = (_bf16(gen, D, std=0.05, mean=1.0) for _ in range(2))
            s.out_k = _bf16(gen, rows, kv, D)
            s.positions = _i32(np.concatenate(
                [p + np.arange(n) for p, n in zip(_past(case), _new(case))] +
                [np.zeros(case["pad"])]))
            if case["cache"]:
                _cache(s, case, gen, seed)
        s.out = _bf16(gen, rows, heads, D)  # rows behind the last sequence keep this
    torch.cuda.synchronize()
    return s


# ---- frequencies ----------------------------------------------------------

BASE, FACTOR, ORIGINAL, LOW, HIGH = 1000000.0, 4.0, 32768.0, 1.0, 32.0


def _frequencies(case):
    """(radians per position [rotary / 2] in 64 bits, factor of the rotated part)"""
    n, how = case["rotary"], case["scaling"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    base = BASE * FACTOR ** (n / (n - 2)) if how == "ntk" else BASE
    f = base ** (-2.0 * i / n)
    if how == "linear":
        f = f / FACTOR
    elif how == "parts":  # by turns over the original length
        keep = ((ORIGINAL * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * keep + f / FACTOR * (1 - keep)
    elif how == "yarn":  # by the pair's place between those of HIGH and LOW turns
        at = [n * math.log(ORIGINAL / (t * 2 * math.pi)) / (2 * math.log(BASE))
              for t in (HIGH, LOW)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
        keep = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * keep + f / FACTOR * (1 - keep)
    return f, 0.1 * math.log(FACTOR) + 1 if how == "yarn" else 1.0


# ---- one pass -------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    kind = s.case["kind"]
    return {"rotary": _plain_rotary, "attention": _plain_attention, "linear": _plain_linear}[kind](s)


def _outputs(s):
    if s.case["kind"] == "rotary":
        return [s.out, s.cache_k, s.cache_v] if s.case["cache"] else [s.out, s.out_k]
    return s.out


def _rotate(x, cos, sin, n, layout):
    """The first n of each head of [rows, heads, D], in 32 bits."""
    if layout == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2),
                      x[..., n:]], -1)


def _plain_rotary(s):
    c = s.case
    heads, kv, used = c["heads"], c["kv_heads"], _rows(c) - c["pad"]
    n = used if c["cache"] else _rows(c)  # without a cache every row is rotated
    f, factor = _frequencies(c)
    angle = s.positions[:n].double()[:, None] * f
    cos, sin = ((t * factor).float()[:, None] for t in (angle.cos(), angle.sin()))
    x = s.qkv[:n].float()
    q, k, v = x[:, :heads], x[:, heads:heads + kv], s.qkv[:n, heads + kv:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s.norm_q.float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s.norm_k.float()
    s.out[:n] = _rotate(q, cos, sin, c["rotary"], c["layout"]).to(torch.bfloat16)
    k = _rotate(k, cos, sin, c["rotary"], c["layout"]).to(torch.bfloat16)
    if c["cache"]:
        row = torch.arange(n, device="cuda")
        seq = torch.searchsorted(s.starts[1:].contiguous(), row.int(), right=True)
        at = s.lengths[seq] - s.starts[seq + 1] + row
        page = s.table[seq, at // c["page"]].long()
        s.cache_k[page, at % c["page"]] = k
        s.cache_v[page, at % c["page"]] = v
    else:
        s.out_k[:n] = k
    return _outputs(s)


def _plain_attention(s):
    c = s.case
    heads, kv, S, Q, T = c["heads"], c["kv_heads"], c["sequences"], s.most, s.longest
    begin, new = s.starts[:-1].long(), (s.starts[1:] - s.starts[:-1]).long()
    i, t = torch.arange(Q, device="cuda"), torch.arange(T, device="cuda")
    live = i < new[:, None]  # [S, Q]
    row = torch.where(live, begin[:, None] + i, 0)
    at = s.lengths[:, None] - new[:, None] + i  # the token's place in its sequence
    page = s.table[:, t // c["page"]].long()  # [S, T]
    there = (page != NO_PAGE) & (t < s.lengths[:, None])
    page = page.clamp(min=0)
    q = s.q[row].float().view(S, Q, kv, heads // kv, D).permute(0, 2, 3, 1, 4).reshape(S, kv, -1, D)
    k = s.cache_k[page, t % c["page"]].float().permute(0, 2, 3, 1).contiguous()  # [S, kv, D, T]
    v = s.cache_v[page, t % c["page"]].float().permute(0, 2, 1, 3).contiguous()
    p = torch.matmul(q, k).view(S, heads, Q, T).mul_(1.0 / math.sqrt(D))
    seen = there[:, None] & (t <= at[..., None])
    if c["window"]:
        seen &= t > at[..., None] - c["window"]
    p.masked_fill_(~seen[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, kv, -1, T), v).view(S, heads, Q, D)
    o = o / torch.where(total > 0, total, 1.0)  # a row that sees nothing is 0
    s.out[row[live]] = o.permute(0, 2, 1, 3)[live].to(torch.bfloat16)
    return _outputs(s)


def _plain_linear(s):
    c = s.case
    q = torch.stack([s.weight & 15, s.weight >> 4], -1).view(c["cols"], -1, c["group"]).float()
    zeros = s.zeros.float()[..., None] if s.zeros is not None else 8.0
    w = ((q - zeros) * s.scales.float()[..., None]).view(c["cols"], c["k"])
    y = torch.matmul(s.x.float(), w.T)
    if s.bias is not None:
        y = y + s.bias.float()
    s.out.copy_(y)
    return _outputs(s)


# ---- the library's calls --------------------------------------------------

_library = None


def _load():
    """(the binding, one context): as a user's program has them."""
    global _library
    if _library is None:
        import importlib.util
        import os
        spec = importlib.util.spec_from_file_location(
            "qdit", os.path.join(os.getcwd(), "qwen-metal_amd", "qdit.py"))
        qd = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(qd)
        _library = qd, qd.Gpu()
    return _library


def _keep(s):
    """The library's handles of the state's tensors and the call's descriptor,
    which a program makes once beside its tensors."""
    import ctypes
    qd, gpu = _load()
    c, handles = s.case, []

    def wrap(t, dtype):
        handles.append(gpu.wrap(t.data_ptr(), t.numel(), dtype) if t is not None else None)
        return handles[-1].h if t is not None else None

    if c["kind"] == "linear":
        d = qd.LinearInt4Desc(
            out=wrap(s.out, qd.BF16), ldc=c["cols"], in_=wrap(s.x, qd.BF16), lda=c["k"],
            weight=wrap(s.weight, qd.I8), scales=wrap(s.scales, qd.BF16),
            zeros=wrap(s.zeros, qd.BF16), bias=wrap(s.bias, qd.BF16), rows=c["rows"], k=c["k"],
            cols=c["cols"], group=c["group"])
        call = qd.lib().qw_gpu_linear_int4
    else:
        heads, kv, rows, cache = c["heads"], c["kv_heads"], _rows(c), None
        if c["kind"] == "attention" or c["cache"]:
            cache = qd.PagedCache(
                k=wrap(s.cache_k, qd.BF16), v=wrap(s.cache_v, qd.BF16),
                table=wrap(s.table, qd.U32), lengths=wrap(s.lengths, qd.U32),
                starts=wrap(s.starts, qd.U32), pages=s.pages, page_size=c["page"],
                table_ld=s.table_ld, sequences=c["sequences"], kv_heads=kv)
            handles.append(cache)
            cache = ctypes.pointer(cache)
        if c["kind"] == "attention":
            d = qd.PagedAttentionDesc(
                out=wrap(s.out, qd.BF16), ldo=heads * D, q=wrap(s.q, qd.BF16), ldq=heads * D,
                cache=cache, rows=rows, heads=heads, head_dim=D, window=c["window"],
                max_new=s.most, max_length=s.longest, scale=1.0 / math.sqrt(D))
            call = qd.lib().qw_gpu_paged_attention_bf16
        else:
            how = {"plain": qd.ROPE_PLAIN, "linear": qd.ROPE_LINEAR, "ntk": qd.ROPE_NTK,
                   "parts": qd.ROPE_BY_PARTS, "yarn": qd.ROPE_YARN}[c["scaling"]]
            turns, factor = qd.rope_turns(rotary_dim=c["rotary"], base=BASE, scaling=how,
                                          factor=FACTOR, original_length=ORIGINAL, low=LOW,
                                          high=HIGH)
            s.turns = torch.from_numpy(turns.view(np.int32)).cuda()
            torch.cuda.synchronize()
            qkv, ld = wrap(s.qkv, qd.BF16), (heads + 2 * kv) * D
            d = qd.RotaryDesc(
                q_out=wrap(s.out, qd.BF16), ldq_out=heads * D, q=qkv, ldq=ld, k=qkv,
                k_offset=heads * D, ldk=ld, rows=rows, heads=heads, kv_heads=kv, head_dim=D,
                positions=wrap(s.positions, qd.U32), turns=wrap(s.turns, qd.U32),
                attention_factor=factor, rotary_dim=c["rotary"],
                layout=qd.ROPE_HALF if c["layout"] == "half" else qd.ROPE_INTERLEAVED, eps=EPS)
            if c["norm"]:
                d.norm_q, d.norm_k = wrap(s.norm_q, qd.BF16), wrap(s.norm_k, qd.BF16)
            if cache:
                d.v, d.v_offset, d.ldv, d.cache = qkv, (heads + kv) * D, ld, cache
            else:
                d.k_out, d.ldk_out = wrap(s.out_k, qd.BF16), kv * D
            call = qd.lib().qw_gpu_rotary_bf16
    return gpu, call, ctypes.byref(d), (d, handles)


def _run_own(s):
    if s.kept is None:
        s.kept = _keep(s)
    gpu, call, desc, _ = s.kept
    if not call(gpu.h, desc):
        raise RuntimeError(gpu.error())
    return _outputs(s)


# ---- what a pass cannot do without ----------------------------------------


def work(case):
    if case["kind"] == "linear":
        n, k, cols = case["rows"], case["k"], case["cols"]
        groups = cols * k // case["group"] * 2
        return {"bytes": cols * k // 2 + groups * (2 if case["zeros"] else 1) +
                2 * n * (k + cols) + 2 * cols * case["bias"],
                "flops": 2 * n * k * cols}
    heads, kv, new = case["heads"], case["kv_heads"], _new(case)
    if case["kind"] == "rotary":
        n = sum(new) + (0 if case["cache"] else case["pad"])
        per = heads + (2 if case["cache"] else 1) * kv  # v only moves with a cache
        return {"bytes": n * (4 * per * D + 4), "flops": n * (heads + kv) * (3 * case["rotary"] + 4 * D)}
    keys = pairs = 0
    w = case["window"] or 1 << 30
    for n, p in zip(new, _past(case)):
        keys += min(p + n, w + n - 1)
        full = max(0, min(n, w - p))  # tokens that see all before them
        pairs += full * p + full * (full + 1) // 2 + (n - full) * w
    return {"bytes": 4 * sum(new) * heads * D + 4 * keys * kv * D, "flops": 4 * heads * D * pairs}


# ---- the same in 64 bits --------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        low, high = (s.weight % 16).double(), (s.weight // 16).double()
        s_, z = s.scales.double(), s.zeros.double() if s.zeros is not None else None
        y = torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        half = case["group"] // 2
        for g in range(case["k"] // case["group"]):
            x = s.x[:, g * 2 * half:(g + 1) * 2 * half].double()
            part = x[:, 0::2] @ low[:, g * half:(g + 1) * half].T
            part += x[:, 1::2] @ high[:, g * half:(g + 1) * half].T
            part -= x.sum(1, keepdim=True) * (z[:, g] if z is not None else 8.0)
            y += part * s_[:, g]
        return y + s.bias.double() if s.bias is not None else y
    return _exact_rotary(s) if case["kind"] == "rotary" else _exact_attention(s)


def _exact_rotary(s):
    c = s.case
    heads, kv, n = c["heads"], c["kv_heads"], c["rotary"]
    rows = _rows(c) - (c["pad"] if c["cache"] else 0)
    turn = []
    for i in range(n // 2):  # radians a position
        f = BASE ** (-2.0 * i / n)
        if c["scaling"] == "linear":
            f /= FACTOR
        elif c["scaling"] == "ntk":
            f = (BASE * FACTOR ** (n / (n - 2))) ** (-2.0 * i / n)
        elif c["scaling"] == "parts":
            turns = ORIGINAL * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - LOW) / (HIGH - LOW)))
            f = keep * f + (1 - keep) * f / FACTOR
        elif c["scaling"] == "yarn":
            first = max(0, math.floor(n / 2 * math.log(ORIGINAL / (HIGH * 2 * math.pi), BASE)))
            last = min(n - 1, math.ceil(n / 2 * math.log(ORIGINAL / (LOW * 2 * math.pi), BASE)))
            keep = 1 - min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = keep * f + (1 - keep) * f / FACTOR
        turn.append(f)
    size = 0.1 * math.log(FACTOR) + 1 if c["scaling"] == "yarn" else 1.0
    angle = s.positions[:rows].double()[:, None] * torch.tensor(turn, dtype=torch.float64,
                                                                device="cuda")
    z = torch.polar(torch.full_like(angle, size), angle)[:, None]

    def turned(x, weight):
        if c["norm"]:
            x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * weight.double()
        y = x.clone()
        if c["layout"] == "half":
            p = torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous()) * z
            y[..., :n // 2], y[..., n // 2:n] = p.real, p.imag
        else:
            p = torch.view_as_complex(x[..., :n].unflatten(-1, (-1, 2)).contiguous()) * z
            y[..., :n] = torch.view_as_real(p).flatten(-2)
        return y

    x = s.qkv[:rows].double()
    q, k = turned(x[:, :heads], s.norm_q), turned(x[:, heads:heads + kv], s.norm_k)
    out = s.out.double()
    out[:rows] = q
    if not c["cache"]:
        out_k = s.out_k.double()
        out_k[:rows] = k
        return [out, out_k]
    ck, cv = s.cache_k.double(), s.cache_v.double()
    table, at = s.table.cpu().numpy(), 0
    for i, (p, m) in enumerate(zip(_past(c), _new(c))):
        t = np.arange(p, p + m)
        page = torch.from_numpy(table[i, t // c["page"]].astype(np.int64)).cuda()
        slot = torch.from_numpy(t % c["page"]).cuda()
        ck[page, slot], cv[page, slot] = k[at:at + m], x[at:at + m, heads + kv:]
        at += m
    return [out, ck, cv]


def _exact_attention(s):
    c = s.case
    G, page = c["heads"] // c["kv_heads"], c["page"]
    out, table, at = s.out.double(), s.table.cpu().numpy(), 0
    for i, (past, n) in enumerate(zip(_past(c), _new(c))):
        t = np.arange(past + n)
        t = t[table[i, t // page] != NO_PAGE]
        where = torch.from_numpy(table[i, t // page].astype(np.int64) * page + t % page).cuda()
        t = torch.from_numpy(t).cuda()
        place = past + torch.arange(n, device="cuda")
        hidden = t[None] > place[:, None]
        if c["window"]:
            hidden |= t[None] + c["window"] <= place[:, None]
        for g in range(c["kv_heads"]):
            k = s.cache_k.view(-1, c["kv_heads"], D)[where, g].double()
            v = s.cache_v.view(-1, c["kv_heads"], D)[where, g].double()
            for h in range(g * G, (g + 1) * G):
                score = s.q[at:at + n, h].double() @ k.T.contiguous() / math.sqrt(D)
                score = score.masked_fill(hidden, -math.inf)
                w = torch.nan_to_num(torch.softmax(score, -1), nan=0.0)
                out[at:at + n, h] = w @ v
        at += n
    return out
