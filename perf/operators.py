"""Measured cases of the 8-bit floating-point expert path and of the router's balance loss.

Four operators: rows of activations quantised to e4m3 with one scale per 128 elements (and gathered into expert order on the way),
the grouped product of such rows with experts stored as e4m3 with one scale per 128 x 128 block, the same product for the gate/up
projection with SiLU(gate) * up quantised in its epilogue, and the balance loss of the router with per-expert counts and its
gradient.  Where ``own`` is false they are computed from elementary torch operations.  Sizes are those of the benchmark
configurations and tests of this repository, with odd and ragged ones beside them.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
E4M3_MAX = 448.0
FLOOR = 2.0 ** -100  # a block's largest magnitude counts as at least this much


# ---- the cases ----------------------------------------------------------------------------------


def _quant(name, tokens, top_k, K):
    return dict(name=name, op="quant", tokens=tokens, top_k=top_k, K=K)


def _gemm(name, op, experts, tokens, top_k, K, N, split="routed", spare=0):
    return dict(name=name, op=op, experts=experts, tokens=tokens, top_k=top_k, K=K, N=N, split=split, spare=spare)


def _balance(name, tokens, experts, top_k, seqs, padded, dtype):
    return dict(name=name, op="balance", tokens=tokens, experts=experts, top_k=top_k, seqs=seqs, padded=padded, dtype=dtype)


def listed():
    return [
        # one sequence being decoded: its hidden state for the eight experts it goes to
        _quant("quant_one_token", 1, 8, 7168),
        # a prefill batch on its way to the experts: every token to eight of them
        _quant("quant_prefill", 4096, 8, 7168),
        # down projection: a prefill batch over 256 experts, about 128 rows each
        _gemm("gemm_prefill", "gemm", 256, 4096, 8, 2048, 7168),
        # projection of a full prefill batch whose tokens crowd on popular experts, some of which get none
        _gemm("gemm_prefill_zipf", "gemm", 256, 8192, 8, 7168, 4096, "zipf"),
        # down projection of a decode step of an odd number of sequences, into a buffer with room for more rows
        _gemm("gemm_decode", "gemm", 256, 37, 8, 2048, 7168, spare=88),
        # down projection of one token: eight experts with one row each
        _gemm("gemm_one_token", "gemm", 256, 1, 8, 2048, 7168),
        # gate/up projection of a prefill batch
        _gemm("gate_up_prefill", "gate_up", 256, 4096, 8, 7168, 4096),
        # gate/up projection of a decode step of 32 sequences
        _gemm("gate_up_decode", "gate_up", 256, 32, 8, 7168, 4096),
        # the smallest call: a few experts of a small model
        _gemm("gate_up_small", "gate_up", 4, 61, 1, 256, 512),
        # the router of a small model during a short fine-tuning step
        _balance("balance_small", 509, 64, 2, 1, 0, "bf16"),
        # one step's tokens over the benchmark's 256 experts, packed sequences of uneven length with padding
        _balance("balance_step", 4096, 256, 8, 7, 61, "bf16"),
        # a long training batch with fp32 router logits
        _balance("balance_long", 65536, 256, 8, 1, 0, "fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, lo, hi, m):
    """A multiple of ``m`` in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, m * int(round(_log_int(rng, lo, hi) / m))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "gate_up", "gate_up", "balance"])
    if op == "quant":
        return dict(op="quant", tokens=_log_int(rng, 1, 4096), top_k=rng.choice([0, 1, 2, 4, 6, 8]), K=_mult(rng, 64, 7168, 16))
    if op == "balance":
        experts = rng.choice([8, 16, 60, 64, 128, 160, 256, 257, 384])
        tokens = _log_int(rng, 1, 65536)
        return dict(op="balance", tokens=tokens, experts=experts, top_k=rng.choice([1, 2, 4, 6, 8]),
                    seqs=_log_int(rng, 1, 64), padded=rng.choice([0, tokens // 16, tokens // 3]), dtype=rng.choice(["bf16", "fp32"]))
    experts = rng.choice([1, 8, 16, 32, 64, 128, 160, 256])
    top_k = rng.choice([k for k in (1, 2, 4, 6, 8) if k <= experts])
    K = _mult(rng, 256, 7168, 16)
    most = min(7168, 7168 * 4096 // K)
    N = _mult(rng, 256, most - most % 256, 256) if op == "gate_up" else _mult(rng, 256, most - most % 16, 16)
    return dict(op=op, experts=experts, tokens=_log_int(rng, 1, 4096), top_k=top_k, K=K, N=N,
                split=rng.choice(["routed", "zipf"]), spare=rng.choice([0, 0, rng.randint(1, 200)]))


# ---- inputs -------------------------------------------------------------------------------------


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


def _e4m3(shape, gen):
    """Normally distributed codes that use the format's range (no NaN codes)."""
    v = torch.randn(shape, generator=gen, device=DEV).mul_(110.0).clamp_(-E4M3_MAX, E4M3_MAX)
    return v.to(torch.float8_e4m3fn).view(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["op"] == "quant":
        T, K, k = case["tokens"], case["K"], case["top_k"]
        x = torch.randn(T, K, generator=gen, device=DEV)
        x *= 1 + 30 * (torch.rand(K, generator=gen, device=DEV) < 0.004)  # a few channels are much larger than the others
        index = None
        if k:  # the token of every row in expert order
            index = torch.randperm(T * k, generator=gen, device=DEV).div(k, rounding_mode="floor").to(torch.int32)
        return dict(op="quant", x=x.to(torch.bfloat16), index=index)
    if case["op"] == "balance":
        T, E, S = case["tokens"], case["experts"], case["seqs"]
        k = min(case["top_k"], E)
        logits = torch.randn(T, E, generator=gen, device=DEV) + 0.5 * torch.randn(E, generator=gen, device=DEV)
        logits = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        idx = logits.float().topk(k, dim=1).indices.to(torch.int32)
        seq_list = mask = None
        if S > 1:  # cumulative ends; the padding behind the last sequence belongs to none
            ends = torch.randint(0, T - case["padded"] + 1, (S,), generator=gen, device=DEV).sort().values
            ends[-1] = T - case["padded"]
            seq_list = ends.to(torch.int64)
        elif case["padded"]:
            mask = torch.ones(T, dtype=torch.bool, device=DEV)
            mask[torch.randperm(T, generator=gen, device=DEV)[: case["padded"]]] = False
        grad = torch.rand(S, generator=gen, device=DEV) + 0.5
        return dict(op="balance", logits=logits.requires_grad_(), idx=idx, seq_list=seq_list, mask=mask, grad=grad)
    G, K, N = case["experts"], case["K"], case["N"]
    counts = _counts(case, gen)
    M = case["tokens"] * case["top_k"] + case["spare"]
    KB, NB = -(-K // BLOCK), -(-N // BLOCK)
    weight = torch.empty(G, K, N, dtype=torch.uint8, device=DEV)
    for g in range(0, G, 16):
        weight[g:g + 16] = _e4m3((min(16, G - g), K, N), gen)
    w_scale = (torch.rand(G, KB, NB, generator=gen, device=DEV) + 0.5) * (K ** -0.5 / 110)
    x = _e4m3((M, K), gen)
    x_scale = (torch.rand(M, KB, generator=gen, device=DEV) + 0.5) * (2.0 / 110)
    s = dict(op=case["op"], x=x, x_scale=x_scale, weight=weight, w_scale=w_scale, counts=counts)
    if case["op"] == "gemm":
        s["out"] = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    else:
        s["out"] = torch.zeros(M, N // 2, dtype=torch.uint8, device=DEV)
        s["out_scale"] = torch.zeros(M, N // 2 // BLOCK, dtype=torch.float32, device=DEV)
    return s


# ---- the plain forms ----------------------------------------------------------------------------


def _quantize(v):
    """Rows of fp32 -> (e4m3 values, scale per 128)."""
    rows, K = v.shape
    b = torch.nn.functional.pad(v, (0, -K % BLOCK)).view(rows, -1, BLOCK)
    a = b.abs().amax(dim=2).clamp(min=FLOOR)
    # 7 * 2^-4 over a * 2^-10 is 448 over a, and neither product is rounded
    code = ((b * 0.4375) / (a * 2.0 ** -10).unsqueeze(2)).to(torch.float8_e4m3fn)
    return code.view(rows, -1)[:, :K].contiguous(), a / E4M3_MAX


def _dequantize(code, scale):
    v = code.view(torch.float8_e4m3fn).float()
    return v * scale.repeat_interleave(BLOCK, dim=-1)[..., :v.shape[-1]]


def _plain_products(s):
    """x[rows of expert g] @ w[g] in fp32, expert by expert (their row counts differ)."""
    row0 = 0
    for g, rows in enumerate(s["counts"].tolist()):
        if rows:
            x = _dequantize(s["x"][row0:row0 + rows], s["x_scale"][row0:row0 + rows])
            w = _dequantize(s["weight"][g], s["w_scale"][g].repeat_interleave(BLOCK, dim=0)[:s["weight"].shape[1]])
            yield row0, row0 + rows, x @ w
        row0 += rows


def _plain_gemm(s):
    out = s["out"].clone()
    for a, b, y in _plain_products(s):
        out[a:b] = y.to(torch.bfloat16)
    return out


def _plain_gate_up(s):
    code, scale = s["out"].view(torch.float8_e4m3fn).clone(), s["out_scale"].clone()
    for a, b, y in _plain_products(s):
        gate, up = y.chunk(2, dim=1)
        code[a:b], scale[a:b] = _quantize(gate / (1 + torch.exp(-gate)) * up)
    return code, scale


def _plain_balance(s):
    logits, idx, S = s["logits"].detach(), s["idx"].long(), s["grad"].numel()
    T, E = logits.shape
    k = idx.shape[1]
    t = torch.arange(T, device=DEV)
    ends = s["seq_list"] if s["seq_list"] is not None else torch.full((1,), T, device=DEV)
    seq = torch.searchsorted(ends, t, right=True)
    used = seq < S if s["mask"] is None else (seq < S) & s["mask"]
    seq = seq.clamp(max=S - 1)
    z = logits.float()
    p = torch.exp(z - z.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True)
    p = p * used.unsqueeze(1)
    n = torch.zeros(S, dtype=torch.float64, device=DEV).index_add_(0, seq, used.double()).clamp(min=1)
    counts = torch.zeros(S, E, dtype=torch.int64, device=DEV)
    counts.view(-1).index_add_(0, (seq.unsqueeze(1) * E + idx).view(-1), used.long().unsqueeze(1).expand(T, k).reshape(-1))
    mean_p = torch.zeros(S, E, dtype=torch.float64, device=DEV).index_add_(0, seq, p.double()) / n.unsqueeze(1)
    f = counts.double() * (E / k) / n.unsqueeze(1)
    loss = (f * mean_p).sum(dim=1).float()
    ft = (f - 1).float()[seq]  # (the 1 cancels in the next line's difference)
    grad = p * (ft - (ft * p).sum(dim=1, keepdim=True)) * (s["grad"] / n.float())[seq].unsqueeze(1)
    return loss, counts, grad.to(logits.dtype)


# ---- one pass -----------------------------------------------------------------------------------


def run(state):
    op = state["op"]
    if not own:
        if op == "quant":
            return _quantize((state["x"] if state["index"] is None else state["x"][state["index"].long()]).float())
        if op == "balance":
            return _plain_balance(state)
        return _plain_gemm(state) if op == "gemm" else _plain_gate_up(state)
    import ascend_kernel_b200 as ak

    if op == "quant":
        code, scale = ak.fp8_quantize_rows(state["x"], state["index"])
        return code.view(torch.float8_e4m3fn), scale
    if op == "balance":
        loss, counts = ak.moe_balance_loss(state["logits"], state["idx"], state["seq_list"], state["mask"])
        (grad,) = torch.autograd.grad(loss, state["logits"], state["grad"])
        return loss.detach(), counts, grad
    args = (state["x"], state["x_scale"], state["weight"], state["w_scale"], state["counts"], state["out"])
    if op == "gemm":
        ak.grouped_gemm_fp8_block(*args, group_list_type=1)
        return state["out"]
    ak.grouped_gemm_fp8_block(*args, output_scale=state["out_scale"], group_list_type=1, gate_up_silu=True)
    return state["out"].view(torch.float8_e4m3fn), state["out_scale"]


# ---- the definitions in 64 bits -----------------------------------------------------------------


def _exact_round_e4m3(v):
    """The nearest e4m3 values: eight steps to a power of two, 2^-9 the smallest, ties to the even one."""
    mantissa, exponent = torch.frexp(v.abs())
    step = torch.exp2(torch.clamp(exponent - 1, min=-6).double() - 3)
    return torch.sign(v) * torch.clamp(torch.round(v.abs() / step) * step, max=E4M3_MAX)


def _exact_quantize(v):
    rows, K = v.shape
    codes = torch.empty(rows, K, dtype=torch.float64, device=DEV)
    scales = []
    for k in range(0, K, BLOCK):
        b = v[:, k:k + BLOCK]
        a = torch.clamp(b.abs().max(dim=1, keepdim=True).values, min=FLOOR)
        codes[:, k:k + BLOCK] = _exact_round_e4m3(b * E4M3_MAX / a)
        scales.append(a / E4M3_MAX)
    return codes, torch.cat(scales, dim=1)


def _e4m3_table():
    c = torch.arange(256, device=DEV)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e.double() - 10))
    v = torch.where((c & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(c >= 128, -v, v)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        x = s["x"].double()
        return _exact_quantize(x if s["index"] is None else x.index_select(0, s["index"]))
    if case["op"] == "balance":
        z = s["logits"].detach().double().requires_grad_()
        T, E = z.shape
        S, k = s["grad"].numel(), s["idx"].shape[1]
        starts = [0] + ([T] if s["seq_list"] is None else s["seq_list"].tolist())
        losses, counts = [], []
        for a, b in zip(starts, starts[1:]):
            p, i = torch.softmax(z[a:b], dim=1), s["idx"][a:b].long()
            if s["mask"] is not None:
                p, i = p[s["mask"][a:b]], i[s["mask"][a:b]]
            c = torch.bincount(i.reshape(-1), minlength=E)
            n = max(1, p.shape[0])
            losses.append(E * torch.dot(c.double() / (k * n), p.sum(dim=0) / n))
            counts.append(c)
        loss = torch.stack(losses)
        (grad,) = torch.autograd.grad(loss, z, s["grad"].double())
        return loss.detach(), torch.stack(counts), grad
    table = _e4m3_table()
    M, K = s["x"].shape
    G, _, N = s["weight"].shape
    kb, nb = torch.arange(K, device=DEV) // BLOCK, torch.arange(N, device=DEV) // BLOCK
    gemm = case["op"] == "gemm"
    out = torch.zeros(M, N if gemm else N // 2, dtype=torch.float64, device=DEV)
    out_scale = None if gemm else torch.zeros(M, N // 2 // BLOCK, dtype=torch.float64, device=DEV)
    row_ends = s["counts"].cumsum(0).tolist()
    for g in range(G):
        a, b = (row_ends[g - 1] if g else 0), row_ends[g]
        if a == b:
            continue
        x = table[s["x"][a:b].long()] * s["x_scale"].double()[a:b][:, kb]
        w = table[s["weight"][g].long()] * s["w_scale"][g].double()[kb][:, nb]
        y = torch.matmul(x, w)
        if gemm:
            out[a:b] = y
        else:
            h = y[:, :N // 2] * torch.sigmoid(y[:, :N // 2]) * y[:, N // 2:]
            out[a:b], out_scale[a:b] = _exact_quantize(h)
    return out if gemm else (out, out_scale)


# ---- what a pass cannot do without ----------------------------------------------------------------


def work(case):
    if case["op"] == "quant":
        T, K = case["tokens"], case["K"]
        rows, KB = T * max(1, case["top_k"]), -(-K // BLOCK)
        return dict(bytes=2 * T * K + rows * (K + 4 * KB) + (4 * rows if case["top_k"] else 0), flops=3 * rows * K)
    if case["op"] == "balance":
        T, E, k = case["tokens"], case["experts"], min(case["top_k"], case["experts"])
        # logits are read for the loss and, once its sums are known, for the gradient
        return dict(bytes=3 * T * E * (2 if case["dtype"] == "bf16" else 4) + 4 * T * k + 12 * case["seqs"] * E, flops=12 * T * E)
    E, T, k, K, N = case["experts"], case["tokens"], case["top_k"], case["K"], case["N"]
    KB, NB = -(-K // BLOCK), -(-N // BLOCK)
    rows = T * k
    active = min(E - E // 64, rows) if case["split"] == "zipf" else E * (1.0 - (1.0 - k / E) ** T)
    result = 2 * N if case["op"] == "gemm" else N // 2 + 4 * (N // 2 // BLOCK)
    return dict(bytes=active * (K * N + 4 * KB * NB) + rows * (K + 4 * KB + result), flops=2 * rows * K * N)
