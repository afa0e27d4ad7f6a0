"""Cases of the operators over the rows of logits (`cuda.logits`): penalties, biases and grammar masks
(`adjust`), the largest entries of a row with its log-sum-exp (`top`), and the distillation loss from a
teacher's top logits with its gradient (`distill_loss`, `distill_grad`, `distill_loss_and_grad`).

`run` computes a case with elementary torch operations, or with the package's kernels where `own` is true."""

import math

import torch

own = False

_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


# ---- the cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one request's decode step: repetition, presence and frequency penalties over a short history
        dict(name="adjust 1 x 32768 float32", op="adjust", rows=1, vocab=32768, dtype="float32", out="float32",
             history=256, bias=0, mask="none", pad=0),
        # a decode batch whose vocabulary is no multiple of anything, in a padded buffer, one grammar for all
        dict(name="adjust 64 x 50021 float16", op="adjust", rows=64, vocab=50021, dtype="float16", out="float16",
             history=2048, bias=16, mask="shared", pad=27),
        # few requests with very long contexts
        dict(name="adjust 8 x 131072 float32, long", op="adjust", rows=8, vocab=131072, dtype="float32",
             out="float32", history=131071, bias=4, mask="none", pad=0),
        # a large decode batch, a grammar per request, float32 for the sampler behind it
        dict(name="adjust 256 x 131072 bfloat16", op="adjust", rows=256, vocab=131072, dtype="bfloat16",
             out="float32", history=4096, bias=64, mask="rows", pad=0),
        # greedy choice of one request's next token
        dict(name="top 1 of 1 x 32768 float32", op="top", rows=1, vocab=32768, dtype="float32", k=1, lse=False,
             temperature=1.0, pad=0),
        # sampling candidates of a decode batch, odd vocabulary
        dict(name="top 50 of 64 x 100003 bfloat16", op="top", rows=64, vocab=100003, dtype="bfloat16", k=50,
             lse=True, temperature=0.75, pad=0),
        # many candidates for few rows: a search over continuations
        dict(name="top 512 of 16 x 131072 float16", op="top", rows=16, vocab=131072, dtype="float16", k=512,
             lse=True, temperature=1.0, pad=0),
        # the teacher's side of distillation over a training batch
        dict(name="top 64 of 4096 x 65536 bfloat16", op="top", rows=4096, vocab=65536, dtype="bfloat16", k=64,
             lse=True, temperature=2.0, pad=0),
        # a short sequence of a small vocabulary
        dict(name="distill loss 16 x 1009 float32", op="loss", rows=16, vocab=1009, dtype="float32",
             teacher="float32", k=8, temperature=1.0, full=False, pad=0),
        # evaluation: the loss alone, the teacher's probabilities over its whole vocabulary
        dict(name="distill loss 2048 x 50021 float16", op="loss", rows=2048, vocab=50021, dtype="float16",
             teacher="float16", k=32, temperature=2.0, full=True, pad=0),
        # the backward pass by itself, after a forward pass that kept the log-sum-exp
        dict(name="distill grad 1024 x 100003 float32", op="grad", rows=1024, vocab=100003, dtype="float32",
             teacher="float32", k=100, temperature=1.0, full=False, pad=0),
        # a training step's loss and gradient together
        dict(name="distill both 4096 x 131072 bfloat16", op="both", rows=4096, vocab=131072, dtype="bfloat16",
             teacher="bfloat16", k=64, temperature=2.0, full=False, pad=0),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["adjust", "top", "loss", "grad", "both"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    items = {"adjust": 1 << 25, "top": 1 << 28, "loss": 1 << 27, "grad": 1 << 27, "both": 1 << 28}[op]
    vocab = _log_uniform(rng, 256, 131072)
    if rng.random() < 0.5:
        vocab |= 1
    vocab = min(vocab, 131072)
    rows = _log_uniform(rng, 1, min(256 if op == "adjust" else 4096, items // vocab))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, pad=rng.choice([0, 0, rng.randint(1, 63)]))
    if op == "adjust":
        case.update(out=rng.choice([dtype, "float32"]), history=_log_uniform(rng, 1, 16384),
                    bias=rng.choice([0, rng.randint(1, 200)]), mask=rng.choice(["none", "shared", "rows"]))
    elif op == "top":
        case.update(k=min(_log_uniform(rng, 1, 1024), vocab), lse=rng.random() < 0.5,
                    temperature=rng.choice([1.0, 0.75, 2.0]))
    else:
        case.update(k=_log_uniform(rng, 1, 200), teacher=rng.choice([dtype, "float32"]),
                    temperature=rng.choice([1.0, 2.0, 4.0]), full=rng.random() < 0.5)
    return case


# ---- inputs ----------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    rows, vocab, pad = case["rows"], case["vocab"], case["pad"]
    dtype = _TORCH[case["dtype"]]
    step = max(1, (1 << 26) // (vocab + pad))        # rows made at a time

    def integers(low, high, shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda")

    def uniforms(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    def normals(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    # rows of a buffer that is `pad` entries wider than the vocabulary
    buffer = torch.empty(rows, vocab + pad, dtype=dtype, device="cuda")
    for at in range(0, rows, step):
        buffer[at:at + step] = normals(min(step, rows - at), vocab + pad).mul_(2.5).to(dtype)
    logits = buffer[:, :vocab]
    state = {"case": case, "logits": logits}
    if case["op"] == "adjust":
        # histories of one token up to `history`, the first row the longest; text repeats few words often
        lengths = integers(1, case["history"] + 1, (rows,))
        lengths[0] = case["history"]
        offsets = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
        offsets[1:] = torch.cumsum(lengths, 0)
        where = uniforms(int(offsets[-1])).pow_(3)
        state["tokens"] = (where * vocab).long().clamp_(max=vocab - 1).to(torch.int32)
        state["offsets"] = offsets
        state["prompts"] = (lengths * uniforms(rows)).long()
        state["repetition"] = 1.0 + 0.25 * uniforms(rows)
        state["presence"] = uniforms(rows)
        state["frequency"] = 0.25 * uniforms(rows)
        if case["bias"]:
            pairs = min(case["bias"], vocab)
            # distinct tokens of a row: one from each of `pairs` equal stretches of the vocabulary
            stretch = vocab // pairs
            picked = torch.arange(pairs, device="cuda")[None, :] * stretch + integers(0, stretch, (rows, pairs))
            state["bias_tokens"] = picked.to(torch.int32).reshape(-1)
            state["bias_values"] = 5.0 * normals(rows * pairs)
            state["bias_offsets"] = torch.arange(rows + 1, device="cuda") * pairs
        if case["mask"] != "none":
            shape = (1 if case["mask"] == "shared" else rows, (vocab + 31) // 32)
            mask = integers(-2 ** 31, 2 ** 31, shape)
            for _ in range(3):                       # a grammar leaves few tokens: one in sixteen
                mask &= integers(-2 ** 31, 2 ** 31, shape)
            if case["mask"] == "rows":
                mask[::2] = -1                       # every other request has no grammar
            state["mask"] = mask.to(torch.int32)
        state["results"] = {"out": torch.empty(rows, vocab, dtype=_TORCH[case["out"]], device="cuda")}
        return state
    if case["op"] == "top":
        state["results"] = {"values": torch.empty(rows, case["k"], dtype=dtype, device="cuda"),
                            "indices": torch.empty(rows, case["k"], dtype=torch.int32, device="cuda")}
        if case["lse"]:
            state["results"]["lse"] = torch.empty(rows, device="cuda")
        return state
    # distinct entries of the vocabulary in any order, values from the largest down
    k = case["k"]
    stretch = vocab // k
    indices = torch.arange(k, device="cuda")[None, :] * stretch + integers(0, stretch, (rows, k))
    indices = torch.gather(indices, 1, torch.argsort(uniforms(rows, k), dim=1))
    values = torch.sort(normals(rows, k).mul_(2.0).add_(8.0), dim=1, descending=True).values
    state["values"] = values.to(_TORCH[case["teacher"]])
    # the student has learnt some of it: its logits are high where the teacher's are
    lift = normals(rows, k).mul_(2.0).add_(5.0)
    logits.scatter_(1, indices, (torch.gather(logits, 1, indices).float() + lift).to(dtype))
    # some rows hold fewer entries, and some positions (padding) none at all
    whole = uniforms(rows)
    counts = torch.where(whole < 0.9, k, integers(1, k + 1, (rows,)))
    counts = torch.where(whole > 0.97, 0, counts)
    absent = torch.arange(k, device="cuda")[None, :] >= counts[:, None]
    state["indices"] = torch.where(absent, -1, indices).to(torch.int32)
    if case["full"]:
        # the teacher's other entries hold 1 to 50 % of its probability
        top = torch.where(absent, -math.inf, state["values"].double() / case["temperature"])
        lse = torch.logsumexp(top, 1) + torch.log1p(uniforms(rows).double() + 0.01)
        state["teacher_lse"] = torch.where(counts > 0, lse, 0.0).float()
    state["grad_loss"] = uniforms(rows) + 0.5
    results = state["results"] = {}
    if case["op"] == "grad":
        state["lse"] = torch.empty(rows, device="cuda")
        for at in range(0, rows, step):
            part = logits[at:at + step].double() / case["temperature"]
            state["lse"][at:at + step] = torch.logsumexp(part, 1).float()
    else:
        results["loss"] = torch.empty(rows, device="cuda")
        results["lse"] = torch.empty(rows, device="cuda")
    if case["op"] != "loss":
        results["out"] = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    return state


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state, state["results"])
    if case["op"] == "adjust":
        return _plain_adjust(case, state)
    if case["op"] == "top":
        return _plain_top(case, state)
    return _plain_distill(case, state)


def _run_own(case, a, r):
    from numba_cuda_amd import logits
    if case["op"] == "adjust":
        logits.adjust(a["logits"], r["out"], tokens=a["tokens"], offsets=a["offsets"], prompt_lengths=a["prompts"],
                      repetition=a["repetition"], presence=a["presence"], frequency=a["frequency"],
                      bias_tokens=a.get("bias_tokens"), bias_values=a.get("bias_values"),
                      bias_offsets=a.get("bias_offsets"), mask=a.get("mask"))
        return r["out"]
    if case["op"] == "top":
        logits.top(a["logits"], case["k"], values=r["values"], indices=r["indices"], lse=r.get("lse"),
                   temperature=case["temperature"])
    elif case["op"] == "loss":
        logits.distill_loss(a["logits"], a["values"], a["indices"], temperature=case["temperature"],
                            teacher_lse=a.get("teacher_lse"), loss=r["loss"], lse=r["lse"])
    elif case["op"] == "grad":
        logits.distill_grad(a["grad_loss"], a["logits"], a["values"], a["indices"], a["lse"],
                            temperature=case["temperature"], teacher_lse=a.get("teacher_lse"), out=r["out"])
    else:
        logits.distill_loss_and_grad(a["grad_loss"], a["logits"], a["values"], a["indices"],
                                     temperature=case["temperature"], teacher_lse=a.get("teacher_lse"),
                                     loss=r["loss"], lse=r["lse"], out=r["out"])
    return r


def _plain_adjust(case, state):
    rows, vocab = case["rows"], case["vocab"]
    x = state["logits"].float()
    tokens, offsets = state["tokens"].long(), state["offsets"]
    place = torch.arange(tokens.numel(), device="cuda")
    row = torch.searchsorted(offsets, place, right=True) - 1
    valid = (tokens >= 0) & (tokens < vocab)
    flat = row * vocab + tokens.clamp(0, vocab - 1)
    made = valid & (place - offsets[row] >= state["prompts"][row])
    seen = torch.zeros(rows * vocab, device="cuda").index_add_(0, flat, valid.float()).view(rows, vocab) > 0
    count = torch.zeros(rows * vocab, device="cuda").index_add_(0, flat, made.float()).view(rows, vocab)
    factor = state["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / factor, x * factor), x)
    x = x - state["frequency"][:, None] * count
    x = x - state["presence"][:, None] * (count > 0)
    if "bias_tokens" in state:
        pair = torch.arange(state["bias_tokens"].numel(), device="cuda")
        row = torch.searchsorted(state["bias_offsets"], pair, right=True) - 1
        bias = torch.zeros(rows * vocab, device="cuda")
        bias[row * vocab + state["bias_tokens"].long()] = state["bias_values"]
        x = x + bias.view(rows, vocab)
    if "mask" in state:
        column = torch.arange(vocab, device="cuda")
        allowed = (state["mask"][:, column >> 5] >> (column & 31)[None, :]) & 1
        x = torch.where(allowed == 1, x, -math.inf)
    return x.to(_TORCH[case["out"]])


def _plain_lse(x, temperature):
    """log sum exp(x / temperature) of the rows of float32 `x`."""
    peak = x.max(dim=1).values
    peak = torch.where(torch.isinf(peak), torch.zeros_like(peak), peak)
    return peak / temperature + torch.log(torch.exp((x - peak[:, None]) / temperature).sum(dim=1))


def _plain_top(case, state):
    logits = state["logits"]
    x = logits.float() + 0.0                         # -0 becomes +0: they are equal
    # a stable sort keeps the lower index first among equal values
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["k"]]
    out = {"values": torch.gather(logits, 1, order), "indices": order.to(torch.int32)}
    if case["lse"]:
        out["lse"] = _plain_lse(x, case["temperature"])
    return out


def _plain_distill(case, state):
    temperature = case["temperature"]
    x = state["logits"].float()
    indices, values = state["indices"].long(), state["values"].float()
    present = (indices >= 0) & (indices < case["vocab"]) & (values > -math.inf)
    at = torch.where(present, indices, torch.zeros_like(indices))
    if case["full"]:
        log_p = values / temperature - state["teacher_lse"][:, None]
    else:
        peak = torch.where(present, values, -math.inf).max(dim=1, keepdim=True).values
        peak = torch.where(torch.isinf(peak), torch.zeros_like(peak), peak)
        log_p = (values - peak) / temperature
        total = torch.where(present, torch.exp(log_p), 0.0).sum(dim=1, keepdim=True)
        log_p = log_p - torch.log(torch.where(total > 0, total, torch.ones_like(total)))
    p = torch.where(present, torch.exp(log_p), 0.0)
    lse = state["lse"] if case["op"] == "grad" else _plain_lse(x, temperature)
    out = {}
    if case["op"] != "grad":
        log_q = torch.gather(x, 1, at) / temperature - lse[:, None]
        out["loss"] = torch.where(p > 0, p * (log_p - log_q), 0.0).sum(dim=1)
        out["lse"] = lse
    if case["op"] != "loss":
        scale = (state["grad_loss"] / temperature)[:, None]
        mass = p.sum(dim=1, keepdim=True)
        grad = scale * mass * torch.exp(x / temperature - lse[:, None])
        grad.scatter_add_(1, at, -scale * p)
        out["out"] = grad.to(state["logits"].dtype)
    return out


# ---- bytes and operations that a pass cannot do without --------------------------------------------

def work(case):
    rows, vocab = case["rows"], case["vocab"]
    size = _BYTES[case["dtype"]]
    items = rows * vocab
    if case["op"] == "adjust":
        # histories are one to `history` tokens long, the first the longest
        tokens = case["history"] + (rows - 1) * (case["history"] + 1) / 2.0
        total = items * (size + _BYTES[case["out"]]) + 4 * tokens + rows * (8 + 8 + 12)
        total += rows * min(case["bias"], vocab) * 8
        if case["mask"] != "none":
            total += (rows if case["mask"] == "rows" else 1) * ((vocab + 31) // 32) * 4
        return {"bytes": total, "flops": 2.0 * tokens}
    if case["op"] == "top":
        total = items * size + rows * case["k"] * (size + 4) + (4 * rows if case["lse"] else 0)
        return {"bytes": total, "flops": items * (4.0 if case["lse"] else 1.0)}
    total = rows * case["k"] * (_BYTES[case["teacher"]] + 4) + items * size + (4 * rows if case["full"] else 0)
    flops = 4.0 * items
    if case["op"] != "grad":
        total += 8 * rows
    if case["op"] != "loss":
        total += items * size + 4 * rows
        flops = 4.0 * items if case["op"] == "grad" else 7.0 * items
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    step = max(1, (1 << 25) // vocab)                # rows in 64 bits at a time
    if case["op"] == "adjust":
        out = torch.empty(rows, vocab, dtype=torch.float64, device="cuda")
        offsets, prompts = state["offsets"].tolist(), state["prompts"].tolist()
        pairs = state["bias_offsets"].tolist() if "bias_tokens" in state else None
        bits = torch.arange(32, device="cuda")
        for r in range(rows):
            line = state["logits"][r].double()
            positive = line > 0
            history = state["tokens"][offsets[r]:offsets[r + 1]].long()
            touched = torch.bincount(history, minlength=vocab) > 0
            made = torch.bincount(history[prompts[r]:], minlength=vocab).double()
            factor = state["repetition"][r].double()
            line[touched & positive] /= factor
            line[touched & ~positive] *= factor
            line -= made * state["frequency"][r].double() + (made > 0).double() * state["presence"][r].double()
            if pairs:
                cut = slice(pairs[r], pairs[r + 1])
                line[state["bias_tokens"][cut].long()] += state["bias_values"][cut].double()
            if "mask" in state:
                words = state["mask"][0 if case["mask"] == "shared" else r].long()
                allowed = ((words[:, None] >> bits[None, :]) & 1).reshape(-1)[:vocab].bool()
                line[~allowed] = -math.inf
            out[r] = line
        return out
    if case["op"] == "top":
        picked = torch.empty(rows, case["k"], dtype=torch.int32, device="cuda")
        lse = torch.empty(rows, dtype=torch.float64, device="cuda")
        for at in range(0, rows, step):
            part = state["logits"][at:at + step]
            # an integer that orders like the value, and below it one that prefers the lower index
            key = (part.float() + 0.0).view(torch.int32).long()
            key = torch.where(key < 0, -(key & 0x7fffffff), key)
            key = key * (1 << 20) + (vocab - 1 - torch.arange(vocab, device="cuda"))
            best = torch.topk(key, case["k"], dim=1).values
            picked[at:at + step] = (vocab - 1 - (best & ((1 << 20) - 1))).to(torch.int32)
            lse[at:at + step] = torch.logsumexp(part.double() / case["temperature"], 1)
        out = {"values": torch.gather(state["logits"], 1, picked.long()).double(), "indices": picked}
        if case["lse"]:
            out["lse"] = lse
        return out
    out = {name: torch.zeros(value.shape, dtype=torch.float64, device="cuda")
           for name, value in state["results"].items()}
    for at in range(0, rows, step):
        cut = slice(at, at + step)
        z = state["logits"][cut].double() / case["temperature"]
        norm = state["lse"][cut].double() if case["op"] == "grad" else torch.logsumexp(z, 1)
        log_q = z - norm[:, None]
        index = state["indices"][cut].long()
        there = index >= 0
        t = torch.where(there, state["values"][cut].double() / case["temperature"], -math.inf)
        if case["full"]:
            total = state["teacher_lse"][cut].double()
        else:
            total = torch.where(there.any(1), torch.logsumexp(t, 1), 0.0)
        log_p = t - total[:, None]
        p = torch.exp(log_p)
        index = torch.where(there, index, 0)
        if case["op"] != "grad":
            term = p * (log_p - torch.gather(log_q, 1, index))
            out["loss"][cut] = torch.where(there, term, 0.0).sum(1)
            out["lse"][cut] = norm
        if case["op"] != "loss":
            grad = p.sum(1)[:, None] * torch.exp(log_q) - torch.zeros_like(z).scatter_add_(1, index, p)
            out["out"][cut] = grad * (state["grad_loss"][cut].double() / case["temperature"])[:, None]
    return out
