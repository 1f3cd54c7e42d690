"""The operators of an attention layer over a paged cache in 4 bits, as cases that can be timed.

  norm       the residual's addition, the root-mean-square norm and its output in 8-bit floating point (e4m3, 1 x 128 blocks with
             an f32 scale): in front of a layer's 8-bit products
  append     the position rotation of new queries and keys, and new keys and values into their sequences' pages in packed 4-bit
             codes with a scale and a bias for each group; followed by the reader, so that what was stored can be seen
  read       cached keys and values of whole sequences out of their pages, as rows of the element type
  attention  softmax attention of new tokens over their sequences' pages: single tokens and prompts

Definitions, for a token at place p of its sequence (the new tokens are the last ones), with query heads sharing a key and value head:

  norm       h = x + r; y = h w / sqrt(mean h^2 + eps); scale = max |y| / 448 over 128 values, code = e4m3(y / scale)
  append     (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) for the pairs of a head's first `rot` values (halves or neighbours),
             with row p of a table; per group: scale = (max - min) / 15 (1 below 1e-7), bias = min,
             code = trunc(clamp((x - bias) (1 / scale) + 0.5, 0, 15)), scale and bias rounded to the element type. The packed
             format has each of these steps rounded to 32 bits: values of few bits lie on the borders between codes often
  read       value = scale code + bias
  attention  out = sum_j softmax_j(scale q . k_j) v_j over j <= p, with a window the last `window` of them
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn
NORM_EPS = 1e-6


def listed():
    return [
        # One token of one stream in front of a projection: nothing but latency.
        dict(name="norm_1_row", op="norm", dtype="bf16", rows=1, cols=4096),
        # A long prompt's rows, the last block of each cut.
        dict(name="norm_5000_rows_f16", op="norm", dtype="f16", rows=5000, cols=4144),
        # The step of a full decode batch.
        dict(name="append_64_tokens", op="append", dtype="bf16", seqs=64, longest=4096, shortest=1, new=1, hq=32, hkv=8, dim=128, group=64, page=16, rot=128, pairs="halves"),
        # Prompts of many lengths at once, half of each head rotated, neighbours paired.
        dict(name="append_prompts_f16", op="append", dtype="f16", seqs=9, longest=2048, shortest=1, new=0, hq=16, hkv=4, dim=128, group=32, page=64, rot=64, pairs="neighbours"),
        # One sequence of moderate length.
        dict(name="read_1000_tokens", op="read", dtype="bf16", seqs=1, longest=1000, shortest=1000, new=0, hkv=8, dim=128, group=64, page=16),
        # Many sequences of odd lengths, moved out whole.
        dict(name="read_many_f16", op="read", dtype="f16", seqs=24, longest=5003, shortest=1, new=0, hkv=8, dim=64, group=32, page=32),
        # One stream's token behind a short conversation: latency.
        dict(name="attention_1_token", op="attention", dtype="bf16", seqs=1, longest=1000, shortest=1000, new=1, hq=32, hkv=8, dim=128, group=64, page=16, window=0),
        # A decode batch over sequences of all lengths: the cache comes from memory.
        dict(name="attention_64_tokens", op="attention", dtype="bf16", seqs=64, longest=8192, shortest=1, new=1, hq=32, hkv=8, dim=128, group=64, page=16, window=0),
        # One stream's token behind a very long document, one scale a head.
        dict(name="attention_far_token_f16", op="attention", dtype="f16", seqs=1, longest=131071, shortest=131071, new=1, hq=32, hkv=8, dim=128, group=128, page=64, window=0),
        # A few drafted tokens a sequence to be checked, in f32, each over a window.
        dict(name="attention_drafts_f32", op="attention", dtype="f32", seqs=12, longest=3001, shortest=40, new=5, hq=16, hkv=8, dim=64, group=32, page=16, window=1024),
        # Prompts of many lengths, some with most of theirs in the cache already.
        dict(name="attention_prompts_f16", op="attention", dtype="f16", seqs=9, longest=2500, shortest=1, new=1100, hq=12, hkv=4, dim=64, group=64, page=32, window=0),
        # A long prompt.
        dict(name="attention_8192_tokens", op="attention", dtype="bf16", seqs=1, longest=8192, shortest=8192, new=0, hq=32, hkv=8, dim=128, group=64, page=16, window=0),
    ]


# What the largest listed cases take: a drawn one takes no more.
MOST_NORMED = 5000 * 4144
MOST_NEW = 64 * 1024 * 128       # keys that come in, by sequence, token, head and value
MOST_CACHED = 64 * 8192 * 8 * 128  # keys of a padded batch
MOST_SCORES = 32 * 8192 * 8192


def _spread(rng, lo, hi, step=1):
    """A whole multiple of `step` from lo to hi, spread over the logarithm."""
    hi = max(lo, hi)
    return min(hi // step * step, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))) / step + 0.5) * step))


def draw(rng):
    op = rng.choice(("norm", "norm", "append", "append", "read", "attention", "attention", "attention", "attention", "attention"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "norm":
        cols = _spread(rng, 256, 16384, 16)
        return dict(op=op, dtype=dtype, rows=_spread(rng, 1, min(8192, MOST_NORMED // cols // (2 if dtype == "f32" else 1))), cols=cols)
    dim = rng.choice((64, 128, 128, 256))
    hkv = rng.choice((1, 2, 4, 8))
    c = dict(op=op, dtype=dtype, hkv=hkv, dim=dim, group=rng.choice([g for g in (32, 64, 64, 128) if g <= dim]), page=rng.choice((16, 16, 32, 64, 256)))
    hq = hkv * rng.choice((1, 2, 3, 4, 4, 8))
    if op == "read":
        seqs = rng.choice((1, _spread(rng, 1, 32)))
        longest = _spread(rng, 16, min(16384, MOST_CACHED // 8 // (seqs * hkv * dim)))
        return dict(c, seqs=seqs, longest=longest, shortest=rng.randint(1, longest), new=0)
    if op == "append":
        c.update(hq=hq, rot=rng.choice((0, dim // 2, dim, dim)), pairs=rng.choice(("halves", "neighbours")))
        if rng.random() < 0.5:
            longest = _spread(rng, 16, 16384)
            return dict(c, seqs=_spread(rng, 1, 128), longest=longest, shortest=rng.randint(1, longest), new=rng.choice((1, 1, rng.randint(2, 8))))
        seqs = rng.choice((1, rng.randint(2, 12)))
        longest = _spread(rng, 16, MOST_NEW // 8 // (seqs * hkv * dim))
        return dict(c, seqs=seqs, longest=longest, shortest=rng.randint(1, longest), new=0)
    c.update(hq=hq, window=rng.choice((0, 0, 0, _spread(rng, 16, 4096))))
    if rng.random() < 0.6:
        seqs, new = rng.choice((1, 1, _spread(rng, 1, 128))), rng.choice((1, 1, 1, rng.randint(2, 8)))
        longest = _spread(rng, 16, min(131072, MOST_CACHED // (seqs * hkv * dim), MOST_SCORES // (seqs * hq * new)))
        return dict(c, seqs=seqs, longest=longest, shortest=rng.choice((longest, rng.randint(1, longest))), new=new)
    seqs = rng.choice((1, rng.randint(2, 10)))
    longest = _spread(rng, 32, min(8192, int(math.sqrt(MOST_SCORES // 2 // (seqs * hq))), MOST_CACHED // 8 // (seqs * hkv * dim)))
    return dict(c, seqs=seqs, longest=longest, shortest=rng.randint(1, longest), new=rng.choice((0, 0, _spread(rng, 9, longest))))


def _lens(c):
    """Tokens of each sequence, the new ones among them, and new tokens of each: the first is the longest, the others are spread evenly in no order."""
    lens = [c["longest"] - int((c["longest"] - c["shortest"]) * (i * 0.6180339887 % 1.0)) for i in range(c["seqs"])]
    if not c["new"]:
        return lens, lens
    return lens, [min(n, c["new"] - int((c["new"] - 1) * (i * 0.7548776662 % 1.0))) for i, n in enumerate(lens)]


def _quantized_into(x, group, dtype):
    """Codes as 32-bit words, scales and biases of x[..., dim], as the cache holds them."""
    x = x.reshape(*x.shape[:-1], -1, group)
    low = x.amin(-1, keepdim=True)
    # A quotient of two tensors: by a plain number torch multiplies with its reciprocal, which rounds twice.
    scale = (x.amax(-1, keepdim=True) - low) / torch.full_like(low, 15.0)
    scale = torch.where(scale < 1e-7, 1.0, scale)
    codes = ((x - low) * (torch.ones_like(scale) / scale) + 0.5).clamp_(0.0, 15.0).to(torch.int32)
    codes = codes.reshape(*codes.shape[:-2], -1, 8) << torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    return codes.sum(-1).to(torch.int32), scale[..., 0].to(dtype), low[..., 0].to(dtype)


def _cosines(positions, rot):
    """A table of cosines and sines, from angles in 64 bits."""
    rate = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * rate
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def prepare(case, seed):
    c, t = case, DTYPES[case["dtype"]]
    gen = torch.Generator("cuda").manual_seed(seed)
    f32, i32 = dict(device="cuda", dtype=torch.float32), dict(device="cuda", dtype=torch.int32)
    s = dict(case=c)

    def normal(*shape):
        return torch.randn(shape, generator=gen, **f32)

    if c["op"] == "norm":
        rows, cols = c["rows"], c["cols"]
        # A residual stream that has grown over its layers, with a few channels far larger than the rest.
        s.update(x=normal(rows, cols).to(t), residual=(4 * normal(rows, cols) * torch.exp(0.5 * normal(cols))).to(t), weight=(1 + 0.2 * normal(cols)).to(t),
                 sum=torch.zeros((rows, cols), device="cuda", dtype=t), codes=torch.zeros((rows, cols), device="cuda", dtype=FP8), scales=torch.zeros((rows, _blocks(cols)), **f32))
        return s
    lens, news = _lens(c)
    seqs, hkv, dim, group, page = c["seqs"], c["hkv"], c["dim"], c["group"], c["page"]
    starts = [sum(news[:i]) for i in range(seqs + 1)]
    tokens, width = starts[-1], -(-max(lens) // page)
    # Pages in the order in which a server comes by them: any. Behind a sequence's last page the table holds no page.
    counts = [-(-n // page) for n in lens]
    order = torch.randperm(sum(counts) + 3, generator=gen, device="cuda").to(torch.int32)
    held = torch.arange(width, device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    pages = torch.full((seqs, width), -1, **i32).masked_scatter_(held, order)
    n_pages = sum(counts) + 3
    seq_of = torch.repeat_interleave(torch.arange(seqs, device="cuda"), torch.tensor(news, device="cuda"))
    first = torch.tensor([n - m for n, m in zip(lens, news)], device="cuda")
    in_seq = torch.arange(tokens, device="cuda") - torch.tensor(starts[:-1], device="cuda")[seq_of]
    s.update(lens=lens, news=news, starts=starts, pages=pages, n_pages=n_pages, offsets=torch.tensor(starts, **i32), held=torch.tensor(lens, **i32), seq_of=seq_of, in_seq=in_seq,
             place_of=first[seq_of] + in_seq)
    for name in ("k", "v"):
        shape = (n_pages, hkv, page, dim)
        if c["op"] == "append":
            s[name + "_codes"] = torch.zeros((*shape[:-1], dim // 8), **i32)
            s[name + "_scales"], s[name + "_biases"] = (torch.zeros((*shape[:-1], dim // group), device="cuda", dtype=t) for _ in range(2))
        else:
            # Keys have an offset to each channel, values have not.
            x = normal(*shape)
            if name == "k":
                x += normal(hkv, 1, dim)
            s[name + "_codes"], s[name + "_scales"], s[name + "_biases"] = _quantized_into(x, group, t)
            del x
    if c["op"] != "read":
        hq = c["hq"]
        wide = (hq + 2 * hkv) * dim if c["op"] == "append" else hq * dim
        # q (, k and v) side by side in a token's row, as the projection leaves them.
        s.update(rows=normal(tokens, wide).to(t), wide=wide, q_out=torch.zeros((tokens, hq, dim), device="cuda", dtype=t))
    if c["op"] in ("append", "read"):
        s.update(k_out=torch.zeros((tokens, hkv, dim), device="cuda", dtype=t), v_out=torch.zeros((tokens, hkv, dim), device="cuda", dtype=t))
    if c["op"] == "append" and c["rot"]:
        s["cos_sin"] = _cosines(max(lens), c["rot"])
    return s


def _blocks(n):
    return (n + 127) // 128


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "append": _own_append, "read": _own_read, "attention": _own_attention}[op](state)
    return {"norm": _plain_norm, "append": _plain_append, "read": _plain_read, "attention": _plain_attention}[op](state)


# ---- the framework's calls


def _framework(c):
    from metaltile_amd import DType, ops
    return {"bf16": DType.BF16, "f16": DType.F16, "f32": DType.F32}[c["dtype"]], ops


def _own_norm(s):
    c = s["case"]
    dt, ops = _framework(c)
    ops.add_rms_norm_fp8(dt, s["x"].data_ptr(), s["residual"].data_ptr(), s["weight"].data_ptr(), NORM_EPS, s["sum"].data_ptr(), s["codes"].data_ptr(), s["scales"].data_ptr(),
                         c["rows"], c["cols"])
    return [s["sum"], s["codes"], s["scales"]]


def _handles(s):
    """The cache and the batch as the framework's calls take them: made once for a state, as a program does."""
    if "cache" not in s:
        c = s["case"]
        _, ops = _framework(c)
        at = lambda n: s[n].data_ptr()  # noqa: E731
        s["cache"] = ops.KvCache(at("k_codes"), at("k_scales"), at("k_biases"), at("v_codes"), at("v_scales"), at("v_biases"), s["n_pages"], c["page"], c["hkv"], c["dim"], c["group"])
        s["batch"] = ops.KvBatch(at("pages"), s["pages"].shape[1], at("held"), len(s["lens"]), s["starts"][-1], max(s["lens"]), offsets=at("offsets"))
    return s["cache"], s["batch"]


def _own_append(s):
    c = s["case"]
    dt, ops = _framework(c)
    cache, batch = _handles(s)
    q, size = s["rows"].data_ptr(), s["rows"].element_size()
    k = q + c["hq"] * c["dim"] * size
    ops.kv_append(dt, cache, batch, k, k + c["hkv"] * c["dim"] * size, row_stride=s["wide"], q=q, q_out=s["q_out"].data_ptr(), hq=c["hq"],
                  cos_sin=s["cos_sin"].data_ptr() if c["rot"] else None, n_positions=max(s["lens"]) if c["rot"] else 0, rot=c["rot"], neighbours=c["pairs"] == "neighbours")
    ops.kv_read(dt, cache, batch, s["k_out"].data_ptr(), s["v_out"].data_ptr())
    return [s["q_out"], s["k_out"], s["v_out"]]


def _own_read(s):
    dt, ops = _framework(s["case"])
    ops.kv_read(dt, *_handles(s), s["k_out"].data_ptr(), s["v_out"].data_ptr())
    return [s["k_out"], s["v_out"]]


def _own_attention(s):
    c = s["case"]
    dt, ops = _framework(c)
    ops.kv_attention(dt, *_handles(s), s["rows"].data_ptr(), s["q_out"].data_ptr(), c["hq"], c["dim"] ** -0.5, window=c["window"])
    return [s["q_out"]]


# ---- the plain forms


def _plain_norm(s):
    c = s["case"]
    rows, cols, blocks = c["rows"], c["cols"], _blocks(c["cols"])
    h = s["x"].float() + s["residual"].float()
    y = h * s["weight"].float() * torch.rsqrt((h * h).mean(1, keepdim=True) + NORM_EPS)
    y = torch.nn.functional.pad(y, (0, -cols % 128)).reshape(rows, blocks, 128)
    most = y.abs().amax(2)
    scales = torch.where(most > 0, most / torch.full_like(most, 448.0), 1.0)
    return [h.to(s["x"].dtype), (y / scales[..., None]).reshape(rows, -1)[:, :cols].to(FP8), scales]


def _slots(s):
    """The page of each new token, and its place there."""
    place, page = s["place_of"], s["case"]["page"]
    return s["pages"][s["seq_of"], place // page].long(), place % page


def _values(s, name, take):
    """Keys or values [..., dim] in 32 bits of what `take` takes of the cache's arrays."""
    words = take(s[name + "_codes"])
    codes = ((words[..., None] >> torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)) & 15).float()
    scales, biases = take(s[name + "_scales"]).float(), take(s[name + "_biases"]).float()
    codes = codes.reshape(*scales.shape, s["case"]["group"])
    return (codes * scales[..., None] + biases[..., None]).reshape(*words.shape[:-1], -1)


def _plain_read(s):
    page, at = _slots(s)
    t = DTYPES[s["case"]["dtype"]]
    return [_values(s, name, lambda x: x[page, :, at]).to(t) for name in ("k", "v")]


def _rotated(x, table, rot, pairs):
    if not rot:
        return x
    half = rot // 2
    cos, sin = table[:, None, :half], table[:, None, half:]
    if pairs == "halves":
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    hq, hkv, dim, rot, t = c["hq"], c["hkv"], c["dim"], c["rot"], s["rows"].dtype
    x = s["rows"].float().reshape(-1, hq + 2 * hkv, dim)
    table = s["cos_sin"][s["place_of"]] if rot else None
    turned = _rotated(x[:, :hq + hkv], table, rot, c["pairs"])
    page, at = _slots(s)
    for name, part in (("k", turned[:, hq:]), ("v", x[:, hq + hkv:])):
        for what, new in zip(("_codes", "_scales", "_biases"), _quantized_into(part, c["group"], t)):
            s[name + what][page, :, at] = new
    return [turned[:, :hq].to(t), *_plain_read(s)]


def _plain_attention(s):
    c = s["case"]
    hq, hkv, dim = c["hq"], c["hkv"], c["dim"]
    seqs, most_new, most = c["seqs"], max(s["news"]), max(s["lens"])
    # All sequences side by side, padded to the longest: [sequence, key head, (query head, new token) or token, value].
    q = torch.zeros((seqs, most_new, hq, dim), device="cuda").index_put_((s["seq_of"], s["in_seq"]), s["rows"].float().reshape(-1, hq, dim))
    q = q.movedim(1, 2).reshape(seqs, hkv, -1, dim)
    pages = s["pages"].clamp_min(0).long()
    k, v = (_values(s, name, lambda x: x[pages].movedim(2, 1).flatten(2, 3)[:, :, :most]) for name in ("k", "v"))
    scores = (q @ k.transpose(-1, -2).contiguous() * dim ** -0.5).reshape(seqs, hq, most_new, most)
    del k
    at = torch.arange(most, device="cuda")
    here = (s["held"].long() - (s["offsets"][1:] - s["offsets"][:-1]))[:, None] + torch.arange(most_new, device="cuda")
    seen = at <= here[..., None]
    if c["window"]:
        seen &= at > here[..., None] - c["window"]
    scores.masked_fill_(~seen[:, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True).reshape(seqs, hkv, -1, 1)
    out = (scores.reshape(seqs, hkv, -1, most) @ v) / total
    out = out.reshape(seqs, hq, most_new, dim)[s["seq_of"], :, s["in_seq"]]
    return [out.to(s["rows"].dtype)]


def _pairs(lens, news, window):
    """Query and key pairs that a head sees."""
    total = 0
    for n, m in zip(lens, news):
        for lo, hi in ((n - m, n),):  # places lo .. hi - 1, each sees min(place + 1, window)
            w = min(window or hi, hi)
            full = max(0, hi - max(lo, w))
            part = hi - lo - full
            total += full * w + part * (2 * lo + part + 1) // 2
    return total


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        return dict(bytes=c["rows"] * c["cols"] * (3 * size + 1) + 4 * c["rows"] * _blocks(c["cols"]) + c["cols"] * size, flops=7.0 * c["rows"] * c["cols"])
    lens, news = _lens(c)
    hkv, dim = c["hkv"], c["dim"]
    cached = 2 * hkv * (dim // 2 + 2 * size * dim // c["group"])  # a token's keys and values in the cache
    if c["op"] == "read":
        return dict(bytes=sum(news) * (cached + 2 * hkv * dim * size), flops=4.0 * sum(news) * hkv * dim)
    hq = c["hq"]
    if c["op"] == "append":
        # rows in, rotated queries out, the cache's share written and what it says of the new tokens
        return dict(bytes=sum(news) * ((2 * hq + 4 * hkv) * dim * size + cached + 4 * c["rot"]), flops=sum(news) * dim * (3.0 * hq + 20.0 * hkv))
    # Every token that some query sees once; four operations for a query, a key and a value of them.
    seen = sum(min(n, c["window"] + m - 1) if c["window"] else n for n, m in zip(lens, news))
    return dict(bytes=sum(news) * 2 * hq * dim * size + seen * cached, flops=4.0 * dim * hq * _pairs(lens, news, c["window"]))


# ---- the definitions in 64 bits


def _e4m3(v):
    """The nearest value of four exponent and three mantissa bits, of two equally near the even one."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(v / step) * step


def _stored64(x, group, dtype):
    """What the cache says of x[tokens, heads, dim]: scales and biases are held in the element type, and a code comes from steps rounded to 32 bits."""
    def r32(v):
        return v.float().double()

    x, out = r32(x), torch.empty_like(x)
    for lo in range(0, x.shape[-1], group):
        part = x[..., lo:lo + group]
        bias, top = part.min(-1)[0], part.max(-1)[0]
        step = r32(r32(top - bias) / 15.0)
        step = torch.where(step < 1e-7, torch.ones_like(step), step)
        code = torch.floor(r32(r32(r32(part - bias[..., None]) * r32(1.0 / step)[..., None]) + 0.5)).clamp(0, 15)
        out[..., lo:lo + group] = step.to(dtype).double()[..., None] * code + bias.to(dtype).double()[..., None]
    return out


def _cached64(s, name, seq, upto):
    """Keys or values [heads, tokens, dim] of a sequence's first tokens."""
    page = s["case"]["page"]
    at = torch.arange(upto, device="cuda")
    rows = s["pages"][seq].long()[at // page]
    words, steps, lows = (s[name + what][rows, :, at % page].movedim(0, 1) for what in ("_codes", "_scales", "_biases"))
    out = torch.empty((*words.shape[:2], s["case"]["dim"]), device="cuda", dtype=torch.float64)
    per = s["case"]["group"]
    for d in range(out.shape[-1]):
        code = words[..., d // 8].long() // 16 ** (d % 8) % 16  # (a floor division: words are signed)
        out[..., d] = steps[..., d // per].double() * code.double() + lows[..., d // per].double()
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        y = s["weight"].double() * h / (h.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
        codes, scales = [], []
        for lo in range(0, c["cols"], 128):
            most = y[:, lo:lo + 128].abs().max(1)[0]
            scale = torch.where(most > 0, most / 448.0, torch.ones_like(most))
            scales.append(scale)
            codes.append(_e4m3(y[:, lo:lo + 128] / scale[:, None]))
        return [h, torch.cat(codes, 1), torch.stack(scales, 1)]
    if c["op"] == "read":
        both = [[_cached64(s, name, i, n).movedim(0, 1) for i, n in enumerate(s["lens"])] for name in ("k", "v")]
        return [torch.cat(x) for x in both]
    t, hkv, dim = DTYPES[c["dtype"]], c["hkv"], c["dim"]
    hq = c["hq"]
    if c["op"] == "append":
        x = s["rows"].double().reshape(-1, hq + 2 * hkv, dim)
        rot = c["rot"]
        if rot:
            row = s["cos_sin"].double()[s["place_of"]]
            for i in range(rot // 2):
                a, b = (i, i + rot // 2) if c["pairs"] == "halves" else (2 * i, 2 * i + 1)
                cos, sin = row[:, i, None], row[:, rot // 2 + i, None]
                one, two = x[:, :hq + hkv, a].clone(), x[:, :hq + hkv, b].clone()
                x[:, :hq + hkv, a] = one * cos - two * sin
                x[:, :hq + hkv, b] = one * sin + two * cos
        return [x[:, :hq], _stored64(x[:, hq:hq + hkv], c["group"], t), _stored64(x[:, hq + hkv:], c["group"], t)]
    out = torch.empty((s["starts"][-1], hq, dim), device="cuda", dtype=torch.float64)
    q = s["rows"].double().reshape(-1, hq, dim)
    shared = hq // hkv
    for i, (n, m) in enumerate(zip(s["lens"], s["news"])):
        k, v = _cached64(s, "k", i, n), _cached64(s, "v", i, n)
        for lo in range(0, m, 1024):
            hi = min(m, lo + 1024)
            here = n - m + torch.arange(lo, hi, device="cuda")[:, None]
            key = torch.arange(n, device="cuda")[None]
            hidden = key > here
            if c["window"]:
                hidden |= key <= here - c["window"]
            rows = slice(s["starts"][i] + lo, s["starts"][i] + hi)
            for h in range(hq):
                p = (q[rows, h] @ k[h // shared].T) / math.sqrt(dim)
                out[rows, h] = torch.softmax(p.masked_fill(hidden, -math.inf), -1) @ v[h // shared]
    return [out]
