"""Measured cases of the way to the experts and back with gradients, and of experts multiplied in 4 bits.

Five operators: the (token, j) pairs sorted by expert from given ids, the rows on their way to the experts and the weighted sum on
their way back (each with its gradient), rows of activations quantised to e2m1 with one power-of-two scale per 32 elements (and gathered
into expert order on the way), and the grouped product of such rows with experts stored the same way, with its gate/up form whose
epilogue quantises SiLU(gate) * up.  Where ``own`` is false they are computed from elementary torch operations.  Sizes are those of the benchmark
configurations and tests of this repository, with odd and ragged ones beside them.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOWEST = -100  # exponent of the smallest scale that quantisation gives a block


# ---- the cases ----------------------------------------------------------------------------------


def _sort(name, tokens, experts, top_k, dropped=0.0):
    return dict(name=name, op="sort", tokens=tokens, experts=experts, top_k=top_k, dropped=dropped)


def _rows(name, op, tokens, experts, top_k, hidden, dtype, dropped=0.0):
    return dict(name=name, op=op, tokens=tokens, experts=experts, top_k=top_k, hidden=hidden, dtype=dtype, dropped=dropped)


def _quant(name, tokens, top_k, K):
    return dict(name=name, op="quant", tokens=tokens, top_k=top_k, K=K)


def _gemm(name, op, experts, tokens, top_k, K, N, split="routed", spare=0):
    return dict(name=name, op=op, experts=experts, tokens=tokens, top_k=top_k, K=K, N=N, split=split, spare=spare)


def listed():
    return [
        # a decode step of an odd number of sequences over the benchmark's 256 experts
        _sort("sort_decode", 37, 256, 8),
        # a long training batch, a few pairs dropped by a capacity
        _sort("sort_long", 65536, 256, 8, 0.03),
        # a short fine-tuning step of a small model in fp32, an odd number of tokens
        _rows("dispatch_small", "dispatch", 509, 64, 2, 2048, "fp32"),
        # one step's tokens on their way to the benchmark's experts
        _rows("dispatch_step", "dispatch", 4096, 256, 8, 7168, "bf16"),
        # the way back of a short step, with pairs dropped and an odd width
        _rows("combine_small", "combine", 509, 64, 2, 1000, "fp32", 0.1),
        # the way back of one step's tokens
        _rows("combine_step", "combine", 4096, 256, 8, 7168, "bf16"),
        # one sequence being decoded: its hidden state for the eight experts it goes to
        _quant("quant_one_token", 1, 8, 7168),
        # a prefill batch on its way to the experts: every token to eight of them
        _quant("quant_prefill", 4096, 8, 7168),
        # down projection: a prefill batch over 256 experts, about 128 rows each
        _gemm("gemm_prefill", "gemm", 256, 4096, 8, 2048, 7168),
        # down projection of a decode step of an odd number of sequences, into a buffer with room for more rows
        _gemm("gemm_decode", "gemm", 256, 37, 8, 2048, 7168, spare=88),
        # gate/up projection of a full prefill batch whose tokens crowd on popular experts, some of which get none
        _gemm("gate_up_prefill_zipf", "gate_up", 256, 8192, 8, 7168, 4096, "zipf"),
        # gate/up projection of one token: eight experts with one row each
        _gemm("gate_up_one_token", "gate_up", 256, 1, 8, 7168, 4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, lo, hi, m):
    """A multiple of ``m`` in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, m * int(round(_log_int(rng, lo, hi) / m))))


def draw(rng):
    op = rng.choice(["sort", "dispatch", "combine", "quant", "gemm", "gemm", "gate_up", "gate_up"])
    if op == "quant":
        return dict(op="quant", tokens=_log_int(rng, 1, 4096), top_k=rng.choice([0, 1, 2, 4, 6, 8]), K=_mult(rng, 64, 7168, 32))
    experts = rng.choice([1, 8, 16, 60, 64, 128, 160, 256] + ([257, 384] if op == "sort" else []))
    top_k = rng.choice([k for k in (1, 2, 4, 6, 8) if k <= experts])
    if op == "sort":
        return dict(op="sort", tokens=_log_int(rng, 1, 65536), experts=experts, top_k=top_k, dropped=rng.choice([0.0, 0.05, 0.4]))
    if op in ("dispatch", "combine"):
        dtype = rng.choice(["bf16", "fp32"])
        hidden = _mult(rng, 64, 7168 if dtype == "bf16" else 3584, 8)
        return dict(op=op, tokens=_log_int(rng, 1, 4096), experts=experts, top_k=top_k, hidden=hidden, dtype=dtype,
                    dropped=rng.choice([0.0, 0.0, 0.1]))
    K = _mult(rng, 256, 7168, 32)
    most = min(7168, 7168 * 4096 // K)
    N = _mult(rng, 256, most - most % 256, 256) if op == "gate_up" else _mult(rng, 256, most - most % 16, 16)
    return dict(op=op, experts=experts, tokens=_log_int(rng, 1, 4096), top_k=top_k, K=K, N=N,
                split=rng.choice(["routed", "zipf"]), spare=rng.choice([0, 0, rng.randint(1, 200)]))


# ---- inputs -------------------------------------------------------------------------------------


def _experts_of(case, gen):
    """The top_k different experts of every token, a share of the pairs dropped (-1)."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    idx = (torch.rand(T, E, generator=gen, device=DEV) + 0.3 * torch.rand(E, generator=gen, device=DEV)).topk(k, dim=1).indices.to(torch.int32)
    if case["dropped"]:
        idx[torch.rand(T, k, generator=gen, device=DEV) < case["dropped"]] = -1
    return idx


def _sorted(idx, E):
    """(token_of, slot) of the pairs in expert order."""
    T, k = idx.shape
    key = torch.where(idx < 0, E, idx).reshape(-1)
    order = key.sort(stable=True).indices
    n = int((key < E).sum())
    token_of = torch.full((T * k,), -1, dtype=torch.int32, device=DEV)
    token_of[:n] = (order[:n] // k).to(torch.int32)
    slot = torch.full((T * k,), -1, dtype=torch.int32, device=DEV)
    slot[order[:n]] = torch.arange(n, dtype=torch.int32, device=DEV)
    return token_of, slot.view(T, k)


def _counts(case, gen):
    """Rows of each expert: every token on top_k different experts, or by popularity (a few experts get none)."""
    E, T, k = case["experts"], case["tokens"], case["top_k"]
    if case["split"] == "zipf":
        p = torch.arange(1, E + 1, dtype=torch.float64, device=DEV).pow(-1.2)[torch.randperm(E, generator=gen, device=DEV)]
        if E >= 64:
            p[torch.randperm(E, generator=gen, device=DEV)[: E // 64]] = 0
        ids = torch.multinomial(p, T * k, replacement=True, generator=gen)
    else:
        ids = torch.rand(T, E, generator=gen, device=DEV).topk(k, dim=1).indices.reshape(-1)
    return torch.bincount(ids, minlength=E).to(torch.int64)


def _codes(v):
    """e2m1 codes of values in units of their scale: nearest, ties to the even code, at most 6."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8)
    for border, even_above in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= border) if even_above else (a > border)
    return c + (torch.signbit(v) * 8).to(torch.uint8)


def _packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _width(K):
    """Bytes of a row of scales: whole words of four."""
    return 4 * -(-K // 128)


def _random_matrix(rows, K, unit, gen):
    """Normally distributed rows in 4 bits: packed codes and scale bytes within a factor of four around ``unit``."""
    codes = torch.empty(rows, K // 2, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // K)
    for r in range(0, rows, step):
        codes[r:r + step] = _packed(_codes(torch.randn(min(step, rows - r), K, generator=gen, device=DEV) * 2))
    middle = 127 + round(math.log2(unit / 2))
    scale = torch.randint(middle - 1, middle + 2, (rows, _width(K)), generator=gen, device=DEV).to(torch.uint8)
    scale[:, K // BLOCK:] = 0
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op = case["op"]
    if op == "sort":
        return dict(op="sort", idx=_experts_of(case, gen), experts=case["experts"])
    if op in ("dispatch", "combine"):
        T, k, H = case["tokens"], case["top_k"], case["hidden"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        token_of, slot = _sorted(_experts_of(case, gen), case["experts"])
        s = dict(op=op, token_of=token_of, slot=slot)
        if op == "dispatch":
            s["x"] = torch.randn(T, H, generator=gen, device=DEV).to(dtype).requires_grad_()
            s["grad"] = torch.randn(T * k, H, generator=gen, device=DEV).to(dtype)
            return s
        s["y"] = torch.randn(T * k, H, generator=gen, device=DEV).to(dtype).requires_grad_()
        s["weight"] = torch.softmax(torch.randn(T, k, generator=gen, device=DEV), dim=1).requires_grad_()
        s["grad"] = torch.randn(T, H, generator=gen, device=DEV).to(dtype)
        return s
    if op == "quant":
        T, K, k = case["tokens"], case["K"], case["top_k"]
        x = torch.randn(T, K, generator=gen, device=DEV)
        x *= 1 + 30 * (torch.rand(K, generator=gen, device=DEV) < 0.004)  # a few channels are much larger than the others
        index = None
        if k:  # the token of every row in expert order
            index = torch.randperm(T * k, generator=gen, device=DEV).div(k, rounding_mode="floor").to(torch.int32)
        return dict(op="quant", x=x.to(torch.bfloat16), index=index)
    G, K, N = case["experts"], case["K"], case["N"]
    counts = _counts(case, gen)
    M = case["tokens"] * case["top_k"] + case["spare"]
    weight, w_scale = _random_matrix(G * N, K, K ** -0.5, gen)
    x, x_scale = _random_matrix(M, K, 2.0, gen)
    s = dict(op=op, x=x, x_scale=x_scale, weight=weight.view(G, N, -1), w_scale=w_scale.view(G, N, -1), counts=counts)
    if op == "gemm":
        s["out"] = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    else:
        s["out"] = torch.zeros(M, N // 4, dtype=torch.uint8, device=DEV)
        s["out_scale"] = torch.zeros(M, N // 2 // BLOCK, dtype=torch.uint8, device=DEV)
    return s


# ---- the plain forms ----------------------------------------------------------------------------


def _plain_sort(s):
    idx, E = s["idx"], s["experts"]
    T, k = idx.shape
    key = torch.where((idx < 0) | (idx >= E), E, idx).reshape(-1)
    at, order = key.sort(stable=True)
    counts = torch.bincount(key, minlength=E + 1)[:E]
    kept = at < E
    token_of = torch.where(kept, order // k, -1).to(torch.int32)
    slot = torch.empty(T * k, dtype=torch.int32, device=DEV)
    slot[order] = torch.where(kept, torch.arange(T * k, device=DEV), -1).to(torch.int32)
    return counts, token_of, slot.view(T, k)


def _plain_dispatch(s):
    x, token_of, slot, g = s["x"].detach(), s["token_of"], s["slot"], s["grad"]
    rows = torch.where((token_of >= 0).unsqueeze(1), x[token_of.clamp(min=0).long()], 0)
    picked = torch.where((slot >= 0).unsqueeze(2), g[slot.clamp(min=0).long()].float(), 0)
    return rows, picked.sum(dim=1).to(x.dtype)


def _plain_combine(s):
    y, w, token_of, slot, g = s["y"].detach(), s["weight"].detach(), s["token_of"], s["slot"], s["grad"].float()
    T, k = slot.shape
    some = (slot >= 0).unsqueeze(2)
    picked = torch.where(some, y[slot.clamp(min=0).long()].float(), 0)
    out = (picked * w.unsqueeze(2)).sum(dim=1).to(y.dtype)
    grad_w = (picked * g.unsqueeze(1)).sum(dim=2)
    w_of = torch.zeros(T * k, device=DEV)  # the weight of every row
    w_of[slot[slot >= 0].long()] = w[slot >= 0]
    grad_y = torch.where((token_of >= 0).unsqueeze(1), g[token_of.clamp(min=0).long()] * w_of.unsqueeze(1), 0)
    return out, grad_y.to(y.dtype), grad_w


def _quantize(v):
    """Rows of fp32 -> (e2m1 codes, exponent of the scale per 32)."""
    rows, K = v.shape
    b = v.view(rows, K // BLOCK, BLOCK)
    a = b.abs().amax(dim=2)
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1): up to 7 units of a power of two, which round to 6
    e = torch.where(m > 0.875, e + 1, e) - 3
    e = torch.where(a > 0, e, LOWEST).clamp(min=LOWEST)
    return _codes(torch.ldexp(b, -e.unsqueeze(2))).view(rows, K), e


def _values(codes, dtype=torch.float32):
    t = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV, dtype=dtype)
    return t[codes.int()]


def _dequantize(packed, scale):
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    K = codes.shape[-1]
    unit = torch.exp2(scale[..., :K // BLOCK].float() - 127)
    return _values(codes) * unit.repeat_interleave(BLOCK, dim=-1)


def _plain_products(s):
    """x[rows of expert g] @ w[g]^T in fp32, expert by expert (their row counts differ)."""
    row0 = 0
    for g, rows in enumerate(s["counts"].tolist()):
        if rows:
            x = _dequantize(s["x"][row0:row0 + rows], s["x_scale"][row0:row0 + rows])
            yield row0, row0 + rows, x @ _dequantize(s["weight"][g], s["w_scale"][g]).T
        row0 += rows


def _plain_gemm(s):
    out = s["out"].clone()
    for a, b, y in _plain_products(s):
        out[a:b] = y.to(torch.bfloat16)
    return out


def _plain_gate_up(s):
    M, I = s["out"].shape[0], 2 * s["out"].shape[1]
    code, scale = torch.zeros(M, I, dtype=torch.uint8, device=DEV), s["out_scale"].clone()
    for a, b, y in _plain_products(s):
        gate, up = y.chunk(2, dim=1)
        code[a:b], e = _quantize(gate / (1 + torch.exp(-gate)) * up)
        scale[a:b] = (e + 127).to(torch.uint8)
    return _values(code, torch.float32).to(torch.float8_e4m3fn), scale.view(torch.float8_e8m0fnu)


# ---- one pass -----------------------------------------------------------------------------------


def _as_e4m3(packed):
    """Packed e2m1 codes as the values they stand for, in a type of 8 bits that has all of them: two bytes for each byte."""
    one = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV).to(torch.float8_e4m3fn).view(torch.uint8).to(torch.int32)
    two = (one.unsqueeze(0) | (one.unsqueeze(1) << 8)).reshape(-1).to(torch.int16)
    return two.index_select(0, packed.reshape(-1).int()).view(torch.float8_e4m3fn).view(packed.shape[0], -1)


def run(state):
    op = state["op"]
    if not own:
        if op == "sort":
            return _plain_sort(state)
        if op == "dispatch":
            return _plain_dispatch(state)
        if op == "combine":
            return _plain_combine(state)
        if op == "quant":
            code, e = _quantize((state["x"] if state["index"] is None else state["x"][state["index"].long()]).float())
            return (_values(code).view(*e.shape, BLOCK) * torch.exp2(e.float()).unsqueeze(2)).view(code.shape).to(torch.bfloat16)
        return _plain_gemm(state) if op == "gemm" else _plain_gate_up(state)
    import ascend_kernel_b200 as ak

    if op == "sort":
        return ak.moe_sort(state["idx"], state["experts"])
    if op == "dispatch":
        rows = ak.moe_dispatch(state["x"], state["token_of"], state["slot"])
        (grad,) = torch.autograd.grad(rows, state["x"], state["grad"])
        return rows.detach(), grad
    if op == "combine":
        out = ak.moe_combine(state["y"], state["weight"], state["token_of"], state["slot"])
        grad_y, grad_w = torch.autograd.grad(out, (state["y"], state["weight"]), state["grad"])
        return out.detach(), grad_y, grad_w
    if op == "quant":  # and read back by the framework's own dequantisation of this format
        code, scale = ak.mxfp4_quantize_rows(state["x"], state["index"])
        rows, K = code.shape[0], 2 * code.shape[1]
        out = torch.empty(rows, K, dtype=torch.bfloat16, device=DEV)
        ak.fp4_dequant(code, scale[:, :K // BLOCK].contiguous(), out)
        return out
    args = (state["x"], state["x_scale"], state["weight"], state["w_scale"], state["counts"], state["out"])
    if op == "gemm":
        ak.grouped_gemm_mxfp4(*args, group_list_type=1)
        return state["out"]
    ak.grouped_gemm_mxfp4(*args, output_scale=state["out_scale"], group_list_type=1, gate_up_silu=True)
    return _as_e4m3(state["out"]), state["out_scale"].view(torch.float8_e8m0fnu)


# ---- the definitions in 64 bits -----------------------------------------------------------------


def _exact_quantize(v):
    """(values in units of the scale, scale): the nearest of the format's numbers, half a unit apart up to 2, then one, then two."""
    rows, K = v.shape
    values, scales = torch.empty_like(v), []
    for k in range(0, K, BLOCK):
        b = v[:, k:k + BLOCK]
        a = b.abs().max(dim=1, keepdim=True).values
        unit = torch.exp2(torch.ceil(torch.log2(torch.clamp(a, min=2.0 ** -140) / 7)).clamp(min=LOWEST))
        unit = torch.where(a > 7 * unit, 2 * unit, torch.where((a <= 3.5 * unit) & (unit > 2.0 ** LOWEST), unit / 2, unit))  # (log2 rounds)
        q = b / unit
        step = torch.where(q.abs() < 2, 0.5, torch.where(q.abs() < 4, 1.0, 2.0))
        values[:, k:k + BLOCK] = torch.clamp(torch.round(q / step) * step, -6, 6)
        scales.append(unit)
    return values, torch.cat(scales, dim=1)


def _exact_values(packed, scale):
    K = 2 * packed.shape[-1]
    k = torch.arange(K, device=DEV)
    c = (packed.index_select(-1, k // 2).long() >> (4 * (k % 2))) & 15
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
    return torch.where(c >= 8, -v, v) * torch.exp2(scale.double() - 127).index_select(-1, k // BLOCK)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sort":
        idx, E = s["idx"].long(), case["experts"]
        T, k = idx.shape
        flat = idx.reshape(-1)
        counts = torch.stack([(flat == e).sum() for e in range(E)])
        start = counts.cumsum(0) - counts
        token_of, slot = torch.full_like(flat, -1), torch.full_like(flat, -1)
        for e in range(E):
            pairs = (flat == e).nonzero().view(-1)
            at = start[e] + torch.arange(pairs.numel(), device=DEV)
            slot[pairs], token_of[at] = at, pairs // k
        return counts, token_of.int(), slot.int().view(T, k)
    if op in ("dispatch", "combine"):
        slot = s["slot"].long()
        T, k = slot.shape
        H, R = case["hidden"], T * k
        g = s["grad"].double()
        if op == "dispatch":
            rows = torch.zeros(R, H, dtype=torch.float64, device=DEV)
            grad = torch.zeros(T, H, dtype=torch.float64, device=DEV)
            for j in range(k):
                t = (slot[:, j] >= 0).nonzero().view(-1)
                rows[slot[t, j]] = s["x"].detach().double()[t]
                grad[t] += g[slot[t, j]]
            return rows, grad
        y, w = s["y"].detach().double(), s["weight"].detach().double()
        out, grad_y, grad_w = torch.zeros(T, H, dtype=torch.float64, device=DEV), torch.zeros_like(y), torch.zeros_like(w)
        for j in range(k):
            t = (slot[:, j] >= 0).nonzero().view(-1)
            r = slot[t, j]
            out[t] += w[t, j, None] * y[r]
            grad_y[r] = w[t, j, None] * g[t]
            grad_w[t, j] = torch.linalg.vecdot(g[t], y[r])
        return out, grad_y, grad_w
    if op == "quant":
        x = s["x"].double()
        values, unit = _exact_quantize(x if s["index"] is None else x.index_select(0, s["index"]))
        return values * unit.index_select(1, torch.arange(case["K"], device=DEV) // BLOCK)
    M, N = s["x"].shape[0], case["N"]
    gemm = op == "gemm"
    out = torch.zeros(M, N if gemm else N // 2, dtype=torch.float64, device=DEV)
    out_scale = None if gemm else torch.full((M, N // 2 // BLOCK), 2.0 ** -127, dtype=torch.float64, device=DEV)
    row_ends = s["counts"].cumsum(0).tolist()
    for g in range(case["experts"]):
        a, b = (row_ends[g - 1] if g else 0), row_ends[g]
        if a == b:
            continue
        y = torch.matmul(_exact_values(s["x"][a:b], s["x_scale"][a:b]), _exact_values(s["weight"][g], s["w_scale"][g]).T)
        if gemm:
            out[a:b] = y
        else:
            out[a:b], out_scale[a:b] = _exact_quantize(y[:, :N // 2] * torch.sigmoid(y[:, :N // 2]) * y[:, N // 2:])
    return out if gemm else (out, out_scale)


# ---- what a pass cannot do without ----------------------------------------------------------------


def work(case):
    op, T = case["op"], case["tokens"]
    if op == "sort":
        pairs = T * case["top_k"]
        return dict(bytes=12 * pairs + 8 * case["experts"], flops=pairs)
    if op in ("dispatch", "combine"):
        pairs, H = T * case["top_k"], case["hidden"]
        size = 2 if case["dtype"] == "bf16" else 4
        # rows one way, their gradients the other
        return dict(bytes=2 * size * (T + pairs) * H + (8 if op == "dispatch" else 16) * pairs, flops=(1 if op == "dispatch" else 5) * pairs * H)
    K = case["K"]
    if op == "quant":
        rows = T * max(1, case["top_k"])
        return dict(bytes=2 * T * K + 2 * rows * K + (4 * rows if case["top_k"] else 0), flops=3 * rows * K)
    E, k, N = case["experts"], case["top_k"], case["N"]
    rows = T * k
    active = min(E - E // 64, rows) if case["split"] == "zipf" else E * (1.0 - (1.0 - k / E) ** T)
    bits = lambda n: n // 2 + n // BLOCK  # noqa: E731
    return dict(bytes=active * N * bits(K) + rows * (bits(K) + (2 * N if op == "gemm" else bits(N // 2))), flops=2 * rows * K * N)
