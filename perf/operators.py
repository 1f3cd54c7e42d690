"""The operators that stand between the packed products of a served model, as cases that can be timed.

  delta     the gated delta rule of a linear-attention layer: q, k, v behind its input projections, in front of the gated
            norm and output projection. One token for each of many sequences, or whole prompts of ragged lengths
  logprobs  log probabilities of given tokens, with the entropy and the top alternatives, behind the output head
  quantize  activations (1 x 128 blocks) and weights (128 x 128 blocks) into 8-bit floating point (e4m3) with an f32 scale
  product   activations times a weight matrix in that format, both ends included: T activations in, T outputs out

Definitions, where a row's block of 128 runs along the last axis and its last block may be shorter:

  delta     S = exp(g) S; u = beta (v - S k); S += u k^T; y = scale S q, for each token in order and each value head;
            q and k over their 2-norms first, sqrt(sum of squares + eps)
  logprobs  x_t - lse, lse = log sum exp x; entropy = lse - sum p x; the largest x in order, of equal ones the lowest index
  quantize  scale = max |x| / 448 over the block (1 for a block of zeros), code = e4m3(x / scale)
  product   out = (codes_x scale_x) (codes_w scale_w)^T
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn
NORM_EPS = 1e-6
CHUNK = 64


def listed():
    return [
        # One stream's token through a small linear-attention layer: nothing but latency.
        dict(name="delta_1_token", op="delta", dtype="bf16", lens="1", hk=16, hv=16, dk=128, dv=128),
        # A full decode batch, two value heads to a key head.
        dict(name="delta_64_sequences", op="delta", dtype="bf16", lens="1x64", hk=16, hv=32, dk=128, dv=128),
        # Prompts of many lengths at once, from a single token on; a length that ends with a chunk and ones that end past it.
        dict(name="delta_ragged_f16", op="delta", dtype="f16", lens="1 2 63 64 65 700 331 17 1024", hk=4, hv=12, dk=64, dv=128),
        # A long prompt.
        dict(name="delta_8192_tokens", op="delta", dtype="bf16", lens="8192", hk=16, hv=32, dk=128, dv=128),
        # One stream's answer: the token taken and five alternatives.
        dict(name="logprobs_1_row", op="logprobs", dtype="bf16", rows=1, vocab=128256, pad=0, top=5, masked=0),
        # A decode batch with f32 logits, tokens banned by -inf, rows of an odd length inside a padded buffer.
        dict(name="logprobs_33_rows_f32", op="logprobs", dtype="f32", rows=33, vocab=50257, pad=47, top=20, masked=1000),
        # A prompt scored whole.
        dict(name="logprobs_4096_rows", op="logprobs", dtype="bf16", rows=4096, vocab=128256, pad=0, top=5, masked=0),
        # A decode batch's activations.
        dict(name="quantize_16_rows", op="quantize", dtype="bf16", rows=16, cols=4096, block=1),
        # A checkpoint's matrix, its last blocks cut both ways.
        dict(name="quantize_weights", op="quantize", dtype="bf16", rows=14300, cols=4144, block=128),
        # One token through an MLP projection: the weights come from memory.
        dict(name="product_1_row", op="product", dtype="bf16", rows=1, n=14336, k=4096),
        # A short prompt of an odd length, f16, an odd number of outputs.
        dict(name="product_77_rows_f16", op="product", dtype="f16", rows=77, n=18943, k=3584),
        # A long prompt through an MLP projection.
        dict(name="product_4096_rows", op="product", dtype="bf16", rows=4096, n=14336, k=4096),
    ]


# What the largest listed cases take: a drawn one takes no more.
MOST_TOKEN_HEADS = 8192 * 32
MOST_LOGITS = 4096 * 128256
MOST_CODES = 14300 * 4144
MOST_MACS = 4096 * 14336 * 4096


def _spread(rng, lo, hi, step=1):
    """A whole multiple of `step` from lo to hi, spread over the logarithm."""
    hi = max(lo, hi)
    return min(hi // step * step, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))) / step + 0.5) * step))


def draw(rng):
    op = rng.choice(("delta", "delta", "delta", "logprobs", "logprobs", "quantize", "product", "product", "product"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "delta":
        hk = rng.choice((2, 4, 8, 16))
        hv = hk * rng.choice((1, 2, 3))
        c = dict(op=op, dtype=dtype, hk=hk, hv=hv, dk=rng.choice((64, 128, 128, 128)), dv=rng.choice((64, 128, 128, 128)))
        if rng.random() < 0.4:
            return dict(c, lens="%dx%d" % (rng.choice((1, 1, 1, rng.randint(2, 8))), _spread(rng, 1, 256)))
        seqs = rng.choice((1, 1, rng.randint(2, 12)))
        most = min(8192, MOST_TOKEN_HEADS // (2 * hv * seqs))
        return dict(c, lens=" ".join(str(_spread(rng, 1 if seqs > 1 else 64, most)) for _ in range(seqs)))
    if op == "logprobs":
        vocab = _spread(rng, 1000, 152064)
        rows = _spread(rng, 1, min(4096, MOST_LOGITS // vocab // (2 if dtype == "f32" else 1)))
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, pad=rng.choice((0, 0, rng.randint(1, 127))), top=rng.choice((0, 1, 5, 20, 32)),
                    masked=rng.choice((0, vocab // 3)))
    if op == "quantize":
        cols = _spread(rng, 128, 16384, 16)
        return dict(op=op, dtype=dtype, rows=_spread(rng, 1, min(16384, MOST_CODES // cols // (2 if dtype == "f32" else 1))), cols=cols, block=rng.choice((1, 1, 128)))
    n, k = _spread(rng, 64, 28672), _spread(rng, 256, 16384, 16)
    return dict(op=op, dtype=dtype, rows=min(rng.choice((1, _spread(rng, 2, 64), _spread(rng, 65, 4096))), MOST_MACS // (n * k)), n=n, k=k)


def _lens(c):
    """Tokens of each sequence: "3 5" or "1x64"."""
    if "x" in c["lens"]:
        length, seqs = map(int, c["lens"].split("x"))
        return [length] * seqs
    return [int(v) for v in c["lens"].split()]


def _blocks(n):
    return (n + 127) // 128


def prepare(case, seed):
    c, t = case, DTYPES[case["dtype"]]
    gen = torch.Generator("cuda").manual_seed(seed)
    f32 = dict(device="cuda", dtype=torch.float32)
    s = dict(case=c)

    def normal(*shape):
        return torch.randn(shape, generator=gen, **f32)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, **f32)

    if c["op"] == "delta":
        lens, hk, hv, dk, dv = _lens(c), c["hk"], c["hv"], c["dk"], c["dv"]
        tokens = sum(lens)
        # What a layer's short convolution leaves, silu of something normal, q, k and v side by side in a token's row.
        width = 2 * hk * dk + hv * dv
        mixed = torch.nn.functional.silu(normal(tokens, width)).to(t)
        # The decay of a state-space layer: a rate of 1..16 for each head times a step of 0.001..0.1 widened by the token.
        rate = 1 + 15 * uniform(hv)
        step = torch.nn.functional.softplus(normal(tokens, hv) + torch.log(torch.expm1(0.001 * 100 ** uniform(hv))))
        starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
        s.update(mixed=mixed, width=width, lens=lens, starts=starts, g=-rate * step, beta=torch.sigmoid(normal(tokens, hv)), state=normal(len(lens), hv, dv, dk) * 0.3,
                 offsets=torch.tensor(starts, device="cuda", dtype=torch.int32), y=torch.zeros((tokens, hv, dv), **f32), state_out=torch.zeros((len(lens), hv, dv, dk), **f32))
        if len(set(lens)) > 1:  # where each sequence's chunks lie in a batch padded to whole ones
            longest = -(-max(lens) // CHUNK) * CHUNK
            s["place"] = torch.tensor([b * longest + i for b, n in enumerate(lens) for i in range(n)], device="cuda")
    elif c["op"] == "logprobs":
        rows, vocab, stride = c["rows"], c["vocab"], c["vocab"] + c["pad"]
        logits = (2.5 * normal(rows, stride)).to(t)
        if c["masked"]:
            logits[:, torch.randperm(vocab, generator=gen, device="cuda")[:c["masked"]]] = -math.inf
        s.update(logits=logits, stride=stride, tokens=torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda", dtype=torch.int32),
                 logprobs=torch.zeros((rows, 1), **f32), entropy=torch.zeros(rows, **f32), top_ids=torch.zeros((rows, c["top"]), device="cuda", dtype=torch.int32),
                 top_logprobs=torch.zeros((rows, c["top"]), **f32))
    elif c["op"] == "quantize":
        rows, cols, block = c["rows"], c["cols"], c["block"]
        x = normal(rows, cols) * (0.05 if block > 1 else torch.exp(normal(rows, 1)))
        s.update(x=x.to(t), codes=torch.zeros((rows, cols), device="cuda", dtype=FP8), scales=torch.zeros((-(-rows // block), _blocks(cols)), **f32))
    else:
        m, n, k = c["rows"], c["n"], c["k"]
        codes = (64 * normal(n, k)).clamp_(-448, 448).to(FP8)
        s.update(w=codes, w_scales=1e-4 * (0.5 + uniform(_blocks(n), _blocks(k))), x=normal(m, k).to(t), out=torch.zeros((m, n), device="cuda", dtype=t))
        if m > 16:
            s.update(x_codes=torch.zeros((m, k), device="cuda", dtype=FP8), x_scales=torch.zeros((m, _blocks(k)), **f32))
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"delta": _own_delta, "logprobs": _own_logprobs, "quantize": _own_quantize, "product": _own_product}[op](state)
    return {"delta": _plain_delta, "logprobs": _plain_logprobs, "quantize": _plain_quantize, "product": _plain_product}[op](state)


# ---- the framework's calls


def _framework(c):
    from metaltile_amd import DType, ops
    return {"bf16": DType.BF16, "f16": DType.F16, "f32": DType.F32}[c["dtype"]], ops


def _own_delta(s):
    c = s["case"]
    dt, ops = _framework(c)
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    q, size = s["mixed"].data_ptr(), s["mixed"].element_size()
    ops.gated_delta_rule(dt, q, q + hk * dk * size, q + 2 * hk * dk * size, s["g"].data_ptr(), s["beta"].data_ptr(), s["state"].data_ptr(), s["state_out"].data_ptr(),
                         s["y"].data_ptr(), len(s["lens"]), s["starts"][-1], hk, hv, dk, dv, row_stride=s["width"], offsets=s["offsets"].data_ptr(), scale=dk ** -0.5,
                         norm_eps=NORM_EPS)
    return [s["y"], s["state_out"]]


def _own_logprobs(s):
    c = s["case"]
    dt, ops = _framework(c)
    ops.token_logprobs(dt, s["logits"].data_ptr(), s["stride"], s["tokens"].data_ptr(), 1, s["logprobs"].data_ptr(), s["entropy"].data_ptr(), s["top_ids"].data_ptr(),
                       s["top_logprobs"].data_ptr(), c["top"], c["rows"], c["vocab"])
    return [s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"]]


def _own_quantize(s):
    c = s["case"]
    dt, ops = _framework(c)
    ops.fp8_quantize(dt, s["x"].data_ptr(), s["codes"].data_ptr(), s["scales"].data_ptr(), c["rows"], c["cols"], c["block"])
    return [s["codes"], s["scales"]]


def _own_product(s):
    c = s["case"]
    dt, ops = _framework(c)
    m, n, k = c["rows"], c["n"], c["k"]
    if m <= 16:
        ops.fp8_qmv(dt, s["w"].data_ptr(), s["w_scales"].data_ptr(), s["x"].data_ptr(), s["out"].data_ptr(), m, n, k)
    else:
        ops.fp8_quantize(dt, s["x"].data_ptr(), s["x_codes"].data_ptr(), s["x_scales"].data_ptr(), m, k, 1)
        ops.fp8_qmm(dt, s["w"].data_ptr(), s["w_scales"].data_ptr(), s["x_codes"].data_ptr(), s["x_scales"].data_ptr(), s["out"].data_ptr(), m, n, k)
    return [s["out"]]


# ---- the plain forms


def _heads(s):
    """q, k (over their 2-norms, a value head each) and v of every token, in 32 bits."""
    c = s["case"]
    hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
    x = s["mixed"].float()
    qk = x[:, :2 * hk * dk].reshape(-1, 2, hk, dk)
    qk = (qk * torch.rsqrt((qk * qk).sum(-1, keepdim=True) + NORM_EPS)).repeat_interleave(hv // hk, 2)
    return qk[:, 0] * dk ** -0.5, qk[:, 1], x[:, 2 * hk * dk:].reshape(-1, hv, dv)


def _plain_delta(s):
    q, k, v = _heads(s)
    g, beta = s["g"], s["beta"]
    seqs, tokens = len(s["lens"]), q.shape[0]
    if max(s["lens"]) == 1:
        S = s["state"] * torch.exp(g)[..., None, None]
        u = beta[..., None] * (v - (S * k[:, :, None]).sum(-1))
        S = S + u[..., None] * k[:, :, None]
        return [(S * q[:, :, None]).sum(-1), S]
    # Sequences side by side, [sequence, head, token, ...], padded to whole chunks by tokens that do nothing.
    padded = -(-max(s["lens"]) // CHUNK) * CHUNK

    def laid(x):
        if "place" in s:
            x = torch.zeros((seqs * padded, *x.shape[1:]), device=x.device).index_copy_(0, s["place"], x)
        else:
            x = torch.nn.functional.pad(x.reshape(seqs, tokens // seqs, -1), (0, 0, 0, padded - tokens // seqs)).reshape(seqs * padded, *x.shape[1:])
        x = x.reshape(seqs, padded // CHUNK, CHUNK, *x.shape[1:])
        return x.movedim(3, 1).contiguous()  # [sequence, head, chunk, token, ...]

    q, k, v, g, beta = (laid(x) for x in (q, k, v, g, beta))
    total = torch.cumsum(g, -1)
    kt = k.transpose(-1, -2).contiguous()
    past = torch.ones((CHUNK, CHUNK), device=q.device).tril().bool()
    decay = torch.exp(torch.where(past, total[..., :, None] - total[..., None, :], -math.inf))
    a = (beta[..., None] * decay * (k @ kt)).tril(-1)
    inside = decay * (q @ kt)
    # (1 + a)^-1 of each chunk, from diagonal blocks of one row to the whole: the inverse of [A 0; C B] is [A' 0; -B' C A' B'].
    inv = torch.eye(CHUNK, device=q.device).expand(a.shape).contiguous()
    size = 1
    while size < CHUNK:
        blocks = a.reshape(*a.shape[:-2], CHUNK // size, size, CHUNK // size, size)
        have = inv.reshape(blocks.shape)
        at = torch.arange(0, CHUNK // size, 2, device=q.device)
        c = blocks[..., at + 1, :, at, :]  # [pair, ..., size, size]
        have[..., at + 1, :, at, :] = -(have[..., at + 1, :, at + 1, :] @ c @ have[..., at, :, at, :])
        size *= 2
    before = torch.exp(total)[..., None]
    u0 = inv @ (beta[..., None] * v)
    w = inv @ (beta[..., None] * before * k)
    qd, left = q * before, torch.exp(total[..., -1:] - total)[..., None]
    kd, last = (k * left).transpose(-1, -2).contiguous(), torch.exp(total[..., -1])[..., None, None]
    S = s["state"].transpose(-1, -2).contiguous()
    y = torch.empty_like(v)
    for i in range(padded // CHUNK):
        u = u0[:, :, i] - w[:, :, i] @ S
        y[:, :, i] = qd[:, :, i] @ S + inside[:, :, i] @ u
        S = last[:, :, i] * S + kd[:, :, i] @ u
    y = y.movedim(1, 3).reshape(seqs, padded, *y.shape[1:2], y.shape[-1])
    y = y.reshape(-1, *y.shape[2:])[s["place"]] if "place" in s else y[:, :tokens // seqs].reshape(tokens, *y.shape[2:])
    return [y, S.transpose(-1, -2).contiguous()]


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"][:, :c["vocab"]].float()
    most = x.amax(1, keepdim=True)
    d = x - most
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total
    logprobs = d.gather(1, s["tokens"].long()) - log_total
    # Of equal logits the lowest index: the logit's bits in their order, and the index's complement below them.
    bits = (x + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + (0xFFFFFFFF - torch.arange(c["vocab"], device=x.device))
    ids = 0xFFFFFFFF - (torch.topk(key, c["top"], dim=1)[0] & 0xFFFFFFFF)
    return [logprobs, entropy[:, 0], ids.int(), d.gather(1, ids) - log_total]


def _quantized(x, block):
    """x in blocks of `block` rows by 128 columns: codes, and a scale for each block."""
    x = x.float()
    rows, cols = x.shape
    padded = torch.nn.functional.pad(x, (0, -cols % 128, 0, -rows % block))
    most = padded.abs().reshape(padded.shape[0] // block, block, padded.shape[1] // 128, 128).amax((1, 3))
    # A quotient of two tensors: by a plain number torch multiplies with its reciprocal, which rounds twice.
    scales = torch.where(most > 0, most / torch.full_like(most, 448.0), 1.0)
    return (x / _per_value(scales, block, rows, cols)).to(FP8), scales


def _per_value(scales, block, rows, cols):
    return scales.repeat_interleave(block, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _plain_quantize(s):
    return list(_quantized(s["x"], s["case"]["block"]))


def _plain_product(s):
    c = s["case"]
    m, n, k = c["rows"], c["n"], c["k"]
    codes, scales = _quantized(s["x"], 1)
    x = codes.float() * _per_value(scales, 1, m, k)
    w = s["w"].float() * _per_value(s["w_scales"], 128, n, k)
    return [(x @ w.T).to(s["x"].dtype)]


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "delta":
        lens = _lens(c)
        hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
        # exp(g) S, S k, the update and S q of every token: one, two, two and two operations for each value of the state.
        return dict(bytes=sum(lens) * ((2 * hk * dk + hv * dv) * size + hv * 8 + hv * dv * 4) + 8 * len(lens) * hv * dv * dk, flops=7.0 * sum(lens) * hv * dk * dv)
    if c["op"] == "logprobs":
        return dict(bytes=c["rows"] * (c["vocab"] * size + 12 + 8 * c["top"]), flops=5.0 * c["rows"] * c["vocab"])
    if c["op"] == "quantize":
        return dict(bytes=c["rows"] * c["cols"] * (size + 1) + 4 * -(-c["rows"] // c["block"]) * _blocks(c["cols"]), flops=3.0 * c["rows"] * c["cols"])
    m, n, k = c["rows"], c["n"], c["k"]
    return dict(bytes=m * k * size + n * k + 4 * _blocks(n) * _blocks(k) + m * n * size, flops=2.0 * m * n * k)


# ---- the definitions in 64 bits


def _e4m3(v):
    """The nearest value of four exponent and three mantissa bits, of two equally near the even one."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(v / step) * step


def _codes64(x, block):
    """Codes' values and scales of x. Scales are held in 32 bits, and what is rounded to a code is a quotient in 32 bits."""
    rows, cols = x.shape
    values, scales = [], []
    for lo in range(0, cols, 128):
        part = x[:, lo:lo + 128].double()
        most = part.abs().amax(1)
        most = torch.nn.functional.pad(most, (0, -rows % block)).reshape(-1, block).amax(1)
        scale = torch.where(most > 0, most / 448.0, torch.ones_like(most)).float().double()
        scales.append(scale)
        values.append(_e4m3((part / scale.repeat_interleave(block)[:rows, None]).float().double()))
    return torch.cat(values, 1), torch.stack(scales, 1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "delta":
        hk, hv, dk, dv = c["hk"], c["hv"], c["dk"], c["dv"]
        x = s["mixed"].double()
        q, k, v = x[:, :hk * dk].reshape(-1, hk, dk), x[:, hk * dk:2 * hk * dk].reshape(-1, hk, dk), x[:, 2 * hk * dk:].reshape(-1, hv, dv)
        q = (q / (q.square().sum(-1, keepdim=True) + NORM_EPS).sqrt() / math.sqrt(dk)).repeat_interleave(hv // hk, 1)
        k = (k / (k.square().sum(-1, keepdim=True) + NORM_EPS).sqrt()).repeat_interleave(hv // hk, 1)
        keep, beta, S = s["g"].double().exp(), s["beta"].double(), s["state"].double()
        y = torch.zeros(v.shape, device="cuda", dtype=torch.float64)
        order = sorted(range(len(s["lens"])), key=lambda b: -s["lens"][b])
        starts = torch.tensor([s["starts"][b] for b in order], device="cuda")
        S = S[order]
        for i in range(max(s["lens"])):  # token i of every sequence that has one: the first ones of that order
            n = sum(length > i for length in s["lens"])
            at = starts[:n] + i
            now = S[:n] * keep[at][..., None, None]
            u = beta[at][..., None] * (v[at] - torch.matmul(now, k[at][..., None])[..., 0])
            now += u[..., None] * k[at][:, :, None]
            y[at] = torch.matmul(now, q[at][..., None])[..., 0]
            S[:n] = now
        out = torch.empty_like(S)
        out[order] = S
        return [y, out]
    if c["op"] == "logprobs":
        logprobs, entropy, top = [], [], []
        for lo in range(0, c["rows"], 256):
            x = s["logits"][lo:lo + 256, :c["vocab"]].double()
            lse = torch.logsumexp(x, 1, keepdim=True)
            p = torch.exp(x - lse)
            logprobs.append(x.gather(1, s["tokens"][lo:lo + 256].long()) - lse)
            entropy.append(-torch.where(p > 0, p * (x - lse), 0.0).sum(1))
            top.append(torch.topk(x, c["top"], dim=1)[0] - lse)
        return [torch.cat(logprobs), torch.cat(entropy), None, torch.cat(top)]
    if c["op"] == "quantize":
        return list(_codes64(s["x"], c["block"]))
    values, scales = _codes64(s["x"], 1)
    x = values * scales.repeat_interleave(128, 1)[:, :c["k"]]
    out = []
    for lo in range(0, c["n"], 4096):
        w = s["w"][lo:lo + 4096].double()
        rows = torch.arange(lo, lo + w.shape[0], device="cuda") // 128
        out.append(x @ (w * s["w_scales"].double()[rows].repeat_interleave(128, 1)[:, :c["k"]]).T)
    return [torch.cat(out, 1)]
