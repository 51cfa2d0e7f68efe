"""What the decode-step operators are measured on: cases, inputs, plain forms and 64-bit forms.

Operators (``helios_b200.ops``):

* ``linear_w4``: projections whose weights are held in 4 bits with group scales;
* ``key_block_bounds``: elementwise key bounds of the 64-key blocks a tick wrote;
* ``sparse_paged_attention``: one query token per row over the key blocks its bounds select;
* ``control_logits``: penalties from a token history, biases and grammar masks on logits.

Layouts (shared by the plain forms and the operators):

* 4-bit weights: ``packed`` int32 ``[N, K / 8]``; word j of a row holds k = 8j .. 8j + 7, the even k's in
  its low 16 bits and the odd k's in its high 16 bits, four bits each in ascending k; ``scales`` bf16
  ``[K / G, N]``, ``zeros`` uint8 ``[K / G, N]`` (8 where there are none).
* bounds of one layer: bf16 ``[pages, Hkv, page / 64, 2, d]`` (minimum, then maximum).
* masks: int32 ``[masks, ceil(V / 32)]``, bit i of word j allows token 32 j + i.
"""

import math

import torch

own = False

BLOCK = 64            # keys per selected block
PAGE = 256            # tokens per KV page
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)  # bit position of k = 8j + i in word j


def listed():
    return [
        # One decoding request: the fused q|k|v projection.
        {"name": "w4 qkv, 1 token", "op": "w4", "m": 1, "k": 2560, "n": 6144, "group": 128, "zeros": False},
        # A small decode batch: the down projection, weights with zero points.
        {"name": "w4 down, 16 tokens", "op": "w4", "m": 16, "k": 9728, "n": 2560, "group": 128, "zeros": True},
        # A decode batch: the fused gate|up projection, finer groups.
        {"name": "w4 gate up, 61 tokens", "op": "w4", "m": 61, "k": 2560, "n": 19456, "group": 64, "zeros": False},
        # A prefill chunk through the same weights.
        {"name": "w4 gate up, 509 tokens", "op": "w4", "m": 509, "k": 2560, "n": 19456, "group": 128, "zeros": True},
        # The bounds' upkeep in a decode tick: one new key per row.
        {"name": "bounds, 64 decode rows", "op": "bounds", "rows": 64, "chunk": 0, "low": 512, "high": 8192,
         "heads": 8, "pages": 2200},
        # The same for a 2048-token prefill chunk beside decode rows.
        {"name": "bounds, 2048-token chunk", "op": "bounds", "rows": 32, "chunk": 2048, "low": 1024, "high": 4096,
         "heads": 8, "pages": 700},
        # One long conversation near the model's context limit.
        {"name": "sparse, 1 row 40k", "op": "sparse", "rows": 1, "low": 40011, "high": 40011, "heads": 8, "group": 4,
         "top": 32},
        # A few requests of very different lengths, some shorter than the budget.
        {"name": "sparse, 16 ragged rows", "op": "sparse", "rows": 16, "low": 500, "high": 40960, "heads": 8,
         "group": 4, "top": 32},
        # A full decode batch of long documents.
        {"name": "sparse, 64 rows", "op": "sparse", "rows": 64, "low": 8192, "high": 20480, "heads": 8, "group": 4,
         "top": 48},
        # One chat request with repetition and frequency penalties.
        {"name": "controls, 1 row", "op": "controls", "rows": 1, "vocab": 151936, "history": 900, "biases": 0,
         "masks": 0},
        # A batch in which some rows follow a grammar and some carry a bias list.
        {"name": "controls, 33 rows", "op": "controls", "rows": 33, "vocab": 151936, "history": 4000, "biases": 300,
         "masks": 8},
        # A full decode batch with long histories and every kind of control.
        {"name": "controls, 128 rows", "op": "controls", "rows": 128, "vocab": 151936, "history": 16000,
         "biases": 64, "masks": 32},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("w4", "bounds", "sparse", "controls"))
    if op == "w4":
        group = rng.choice((32, 64, 128))
        k = group * _log(rng, 2, 9728 // group)
        n = _log(rng, 60, 19456)
        m = _log(rng, 1, 1024)
        m = max(1, min(m, 509 * 2560 * 19456 // (k * n)))
        return {"op": op, "m": m, "k": k, "n": n, "group": group, "zeros": rng.random() < 0.5}
    if op == "bounds":
        high = _log(rng, 300, 8192)
        rows = _log(rng, 1, 64)
        chunk = rng.choice((0, _log(rng, 17, 2048)))
        return {"op": op, "rows": rows, "chunk": chunk, "low": rng.randint(1, high), "high": high,
                "heads": rng.choice((2, 4, 8)), "pages": 2200}
    if op == "sparse":
        high = _log(rng, 100, 40960)
        rows = max(1, min(_log(rng, 1, 64), 64 * 14336 // high))
        return {"op": op, "rows": rows, "low": rng.randint(1, high), "high": high, "heads": rng.choice((2, 4, 8)),
                "group": rng.choice((1, 2, 4, 8)), "top": rng.randint(4, 48)}
    return {"op": op, "rows": _log(rng, 1, 128), "vocab": _log(rng, 1000, 151936), "history": _log(rng, 1, 16000),
            "biases": rng.choice((0, _log(rng, 1, 300))), "masks": rng.choice((0, rng.randint(1, 32)))}


# ---------------------------------------------------------------- inputs
def _generators(seed):
    gpu = torch.Generator(device="cuda")
    gpu.manual_seed(seed)
    cpu = torch.Generator()
    cpu.manual_seed(seed)
    return gpu, cpu


def prepare(case, seed):
    gpu, cpu = _generators(seed)
    state = {"case": case}
    state.update({"w4": _prepare_w4, "bounds": _prepare_bounds, "sparse": _prepare_sparse,
                  "controls": _prepare_controls}[case["op"]](case, gpu, cpu))
    return state


def _prepare_w4(case, gpu, cpu):
    m, k, n, group = case["m"], case["k"], case["n"], case["group"]
    x = torch.randn(m, k, generator=gpu, device="cuda")
    x[:, ::97] *= 6  # a few channels carry most of a hidden state's energy
    code = (torch.randn(n, k, generator=gpu, device="cuda") * 2.6 + 8).round_().clamp_(0, 15).to(torch.int32)
    code = code.view(n, k // 8, 8)
    packed = torch.zeros(n, k // 8, dtype=torch.int32, device="cuda")
    for i, shift in enumerate(SHIFTS):
        packed |= code[:, :, i] << shift
    scales = (torch.rand(k // group, n, generator=gpu, device="cuda") * 0.01 + 0.004).to(torch.bfloat16)
    zeros = (torch.randint(5, 12, (k // group, n), generator=gpu, device="cuda", dtype=torch.uint8)
             if case["zeros"] else None)
    return {"x": x.to(torch.bfloat16), "packed": packed, "scales": scales, "zeros": zeros}


def _lengths(case, cpu):
    return torch.randint(case["low"], case["high"] + 1, (case["rows"],), generator=cpu).tolist()


def _pages(lengths, cpu, total):
    """A block table over shuffled pages (int32 ``[rows, width]``, zero-padded)."""
    need = [-(-length // PAGE) for length in lengths]
    order = torch.randperm(total, generator=cpu)[:sum(need)].tolist()
    table = torch.zeros(len(lengths), max(need), dtype=torch.int32)
    at = 0
    for row, count in enumerate(need):
        table[row, :count] = torch.tensor(order[at:at + count], dtype=torch.int32)
        at += count
    return table


def _keys(pages, heads, gpu):
    """Keys whose blocks differ in direction and whose channels differ in size, as a model's do."""
    keys = torch.randn(pages, PAGE, heads, 128, generator=gpu, device="cuda", dtype=torch.bfloat16)
    drift = torch.randn(pages, PAGE // BLOCK, 1, heads, 128, generator=gpu, device="cuda", dtype=torch.bfloat16)
    keys.view(pages, PAGE // BLOCK, BLOCK, heads, 128).add_(drift)
    keys[..., 5] *= 4
    keys[..., 70] *= 4
    return keys


def _prepare_bounds(case, gpu, cpu):
    lengths, counts = _lengths(case, cpu), [1] * case["rows"]
    if case["chunk"]:
        lengths, counts = lengths + [case["chunk"] + 37], counts + [case["chunk"]]
    need = sum(-(-length // PAGE) for length in lengths)
    pages = max(case["pages"], need)
    table = _pages(lengths, cpu, pages)
    cu = torch.tensor([0] + counts).cumsum(0)
    token_row = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    keys = _keys(pages, case["heads"], gpu)
    bounds = torch.zeros(pages, case["heads"], PAGE // BLOCK, 2, 128, dtype=torch.bfloat16, device="cuda")
    starts = [length - count for length, count in zip(lengths, counts)]
    blocks = [(row, block) for row, (start, length) in enumerate(zip(starts, lengths))
              for block in range(start // BLOCK, (length - 1) // BLOCK + 1)]
    return {"keys": keys, "bounds": bounds, "table": table.cuda(), "cu": cu.int().cuda(),
            "used": torch.tensor(lengths, dtype=torch.int32).cuda(), "token_row": token_row.int().cuda(),
            "blocks": torch.tensor(blocks).cuda()}


def _prepare_sparse(case, gpu, cpu):
    lengths = _lengths(case, cpu)
    heads, group = case["heads"], case["group"]
    pages = sum(-(-length // PAGE) for length in lengths) + 3
    table = _pages(lengths, cpu, pages)
    keys = _keys(pages, heads, gpu)
    values = torch.randn(pages, PAGE, heads, 128, generator=gpu, device="cuda", dtype=torch.bfloat16)
    blocks = keys.view(pages, PAGE // BLOCK, BLOCK, heads, 128)
    bounds = torch.stack((blocks.amin(2), blocks.amax(2)), dim=3).permute(0, 2, 1, 3, 4).contiguous()
    q = torch.randn(len(lengths), heads * group, 128, generator=gpu, device="cuda").to(torch.bfloat16)
    return {"q": q, "keys": keys, "values": values, "bounds": bounds, "table": table.cuda(),
            "used": torch.tensor(lengths, dtype=torch.int32).cuda(), "max_blocks": -(-max(lengths) // BLOCK)}


def _prepare_controls(case, gpu, cpu):
    rows, vocab, most = case["rows"], case["vocab"], case["history"]
    logits = (torch.randn(rows, vocab, generator=gpu, device="cuda") * 3).to(torch.bfloat16)
    # Histories of very different lengths in a wider arena; text repeats a few tokens often.
    slots = torch.randperm(rows + 5, generator=cpu)[:rows].int()
    lengths = torch.randint(0, most + 1, (rows + 5,), generator=cpu).int()
    lengths[slots[0].long()] = most
    prompts = (lengths * torch.rand(rows + 5, generator=cpu)).int()
    skew = torch.rand(rows + 5, most, generator=gpu, device="cuda") ** 4
    state = {"logits": logits, "history": (skew * vocab).int().clamp_(0, vocab - 1), "slots": slots.cuda(),
             "lengths": lengths.cuda(), "prompts": prompts.cuda(),
             "repetition": (1 + torch.rand(rows, generator=cpu) * 0.3).cuda(),
             "frequency": (torch.rand(rows, generator=cpu) * 0.5).cuda(),
             "presence": (torch.rand(rows, generator=cpu) * 0.8 - 0.2).cuda(),
             "bias": None, "mask": None, "mask_rows": None}
    if case["biases"]:
        counts = torch.randint(0, min(case["biases"], vocab // 2) + 1, (rows,), generator=cpu)
        tokens = [torch.randperm(vocab, generator=cpu)[:c].sort().values for c in counts.tolist()]
        tokens = torch.cat(tokens).int()
        values = torch.randn(tokens.numel(), generator=cpu) * 4
        values[::5] = -100.0  # tokens that the request bans
        offsets = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0))).int()
        state["bias"] = (offsets.cuda(), tokens.cuda(), values.cuda())
    if case["masks"]:
        words = -(-vocab // 32)
        draws = [torch.randint(-2 ** 31, 2 ** 31 - 1, (case["masks"], words), generator=gpu, device="cuda",
                               dtype=torch.int64).int() for _ in range(4)]
        state["mask"] = draws[0] & draws[1] & draws[2] & draws[3]  # a grammar allows a small part
        pick = torch.randint(0, case["masks"], (rows,), generator=cpu)
        pick[torch.rand(rows, generator=cpu) < 0.4] = -1  # rows without a grammar
        state["mask_rows"] = pick.int().cuda()
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        from helios_b200 import ops
        if case["op"] == "w4":
            return ops.linear_w4(state["x"], state["packed"], state["scales"], state["zeros"])
        if case["op"] == "bounds":
            return ops.key_block_bounds(state["keys"], state["bounds"], state["table"], state["cu"], state["used"],
                                        state["token_row"])
        if case["op"] == "sparse":
            selected = torch.empty(case["rows"], case["heads"], case["top"], dtype=torch.int32, device="cuda")
            out = ops.sparse_paged_attention(state["q"], state["keys"], state["values"], state["bounds"],
                                             state["table"], state["used"], top_blocks=case["top"],
                                             selected=selected)
            return {"out": out, "selected": selected}
        return ops.control_logits(state["logits"], repetition=state["repetition"], frequency=state["frequency"],
                                  presence=state["presence"], history=state["history"], slots=state["slots"],
                                  lengths=state["lengths"], prompt_lengths=state["prompts"], bias=state["bias"],
                                  mask=state["mask"], mask_rows=state["mask_rows"])
    return {"w4": _plain_w4, "bounds": _plain_bounds, "sparse": _plain_sparse,
            "controls": _plain_controls}[case["op"]](state)


def _plain_w4(state):
    packed, scales, zeros = state["packed"], state["scales"], state["zeros"]
    n, k = packed.shape[0], packed.shape[1] * 8
    shifts = torch.tensor(SHIFTS, dtype=torch.int32, device=packed.device)
    code = ((packed.unsqueeze(-1) >> shifts) & 15).view(n, scales.shape[0], -1).float()
    zero = 8.0 if zeros is None else zeros.t().unsqueeze(-1).float()
    weight = ((code - zero) * scales.t().unsqueeze(-1).float()).view(n, k)
    return (state["x"].float() @ weight.t()).to(torch.bfloat16)


def _plain_bounds(state):
    keys, bounds, table, used = state["keys"], state["bounds"], state["table"], state["used"]
    rows, blocks = state["blocks"][:, 0], state["blocks"][:, 1]
    per_page = PAGE // BLOCK
    pages, at = table[rows, blocks // per_page].long(), blocks % per_page
    part = keys.view(keys.shape[0], per_page, BLOCK, keys.shape[2], 128)[pages, at].float()
    position = blocks.unsqueeze(1) * BLOCK + torch.arange(BLOCK, device=keys.device)
    outside = (position >= used[rows].unsqueeze(1)).view(-1, BLOCK, 1, 1)
    low = part.masked_fill(outside, math.inf).amin(1)
    high = part.masked_fill(outside, -math.inf).amax(1)
    bounds[pages, :, at] = torch.stack((low, high), dim=2).to(torch.bfloat16)
    return bounds


def _plain_sparse(state):
    q, keys, values, table, used = state["q"], state["keys"], state["values"], state["table"], state["used"]
    top, per_page, device = state["case"]["top"], PAGE // BLOCK, q.device
    rows, heads = q.shape[0], keys.shape[2]
    group = q.shape[1] // heads
    blocks = torch.arange(state["max_blocks"], device=device)
    at = table[:, blocks // per_page].long() * per_page + blocks % per_page           # [rows, blocks]
    count = (used.long() + BLOCK - 1) // BLOCK
    # Scores in 64 bits: two implementations have to agree on which of two close blocks is larger.
    bounds = state["bounds"].transpose(1, 2).reshape(-1, heads, 2, 128)[at].double()   # [rows, blocks, heads, 2, d]
    part = q.view(rows, heads, group, 128).double()
    score = (torch.einsum("rhgd,rbhd->rhgb", part.clamp(max=0), bounds[:, :, :, 0])
             + torch.einsum("rhgd,rbhd->rhgb", part.clamp(min=0), bounds[:, :, :, 1])).amax(2)
    last = count.view(-1, 1, 1)
    forced = (blocks < 1) | (blocks >= last - 2)
    score = score.masked_fill(forced, math.inf).masked_fill(blocks >= last, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[:, :, :top]
    chosen = order.masked_fill(order >= last, state["max_blocks"]).sort(dim=-1).values
    if chosen.shape[2] < top:
        chosen = torch.nn.functional.pad(chosen, (0, top - chosen.shape[2]), value=state["max_blocks"])
    empty = chosen >= last
    where = at.unsqueeze(1).expand(-1, heads, -1).gather(2, chosen.clamp(max=state["max_blocks"] - 1))
    head = torch.arange(heads, device=device).view(1, -1, 1)
    k = keys.view(-1, BLOCK, heads, 128)[where, :, head].float().flatten(2, 3)         # [rows, heads, top * 64, d]
    v = values.view(-1, BLOCK, heads, 128)[where, :, head].float().flatten(2, 3)
    position = chosen.unsqueeze(-1) * BLOCK + torch.arange(BLOCK, device=device)
    outside = (empty.unsqueeze(-1) | (position >= used.view(-1, 1, 1, 1))).flatten(2).unsqueeze(2)
    s = (part.float() @ k.transpose(2, 3) * 128 ** -0.5).masked_fill(outside, -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    out = p @ v / p.sum(-1, keepdim=True)
    return {"out": out.view(rows, heads * group, 128).to(torch.bfloat16),
            "selected": chosen.masked_fill(empty, -1).int()}


def _plain_controls(state):
    logits, slots = state["logits"], state["slots"].long()
    rows, vocab = logits.shape
    x = logits.float()
    history = state["history"][slots].long()
    position = torch.arange(history.shape[1], device=x.device)
    told = position < state["lengths"][slots].unsqueeze(1)
    prompt = position < state["prompts"][slots].unsqueeze(1)
    seen = torch.zeros_like(x).scatter_add_(1, history, told.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, history, (told & ~prompt).float())
    r = state["repetition"].unsqueeze(1)
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - state["frequency"].unsqueeze(1) * count
    x = x - state["presence"].unsqueeze(1) * (count > 0)
    if state["bias"] is not None:
        offsets, tokens, values = state["bias"]
        at = torch.arange(tokens.numel(), device=x.device)
        row = torch.searchsorted(offsets, at, right=True, out_int32=False) - 1
        x = x.index_put((row, tokens.long()), values, accumulate=True)
    if state["mask"] is not None:
        token = torch.arange(vocab, device=x.device)
        words = state["mask"][state["mask_rows"].long().clamp(min=0)][:, token // 32]
        banned = ((words >> (token % 32)) & 1) == 0
        x = x.masked_fill(banned & (state["mask_rows"] >= 0).unsqueeze(1), -math.inf)
    return x.to(torch.bfloat16)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "w4":
        m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
        return {"bytes": n * k // 2 + n * groups * (3 if case["zeros"] else 2) + 2 * m * (k + n), "flops": 2 * m * n * k}
    if case["op"] == "bounds":
        # Half a block of each decode row's last block on average, the whole chunk; two rows written per block.
        keys = case["rows"] * BLOCK // 2 + case["chunk"]
        blocks = case["rows"] + -(-case["chunk"] // BLOCK)
        return {"bytes": 256 * case["heads"] * (keys + 2 * blocks), "flops": 2 * 128 * case["heads"] * keys}
    if case["op"] == "sparse":
        mean = (case["low"] + case["high"]) / 2
        blocks = mean / BLOCK
        chosen = min(blocks, case["top"])
        pairs = case["rows"] * case["heads"]
        return {"bytes": pairs * (blocks * 512 + chosen * BLOCK * 512 + case["group"] * 512),
                "flops": pairs * case["group"] * (blocks * 512 + chosen * BLOCK * 512)}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (4 * vocab + 2 * case["history"] + 4 * case["biases"]) + case["masks"] * vocab // 8,
            "flops": 2 * rows * vocab}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"w4": _exact_w4, "bounds": _exact_bounds, "sparse": _exact_sparse,
            "controls": _exact_controls}[case["op"]](state)


def _exact_w4(state):
    packed, scales, zeros, x = state["packed"], state["scales"], state["zeros"], state["x"].double()
    groups, n = scales.shape
    words = packed.shape[1] // groups
    out = torch.zeros(x.shape[0], n, dtype=torch.float64, device=x.device)
    for g in range(groups):
        for i, shift in enumerate(SHIFTS):
            q = ((packed[:, g * words:(g + 1) * words] >> shift) & 15).double()
            q -= 8 if zeros is None else zeros[g].double().unsqueeze(1)
            start = g * words * 8 + i
            out += scales[g].double() * (x[:, start:start + 8 * words:8] @ q.t())
    return out


def _exact_bounds(state):
    bounds, keys, used = state["bounds"].double(), state["keys"], state["used"].tolist()
    table = state["table"].tolist()
    for row, block in state["blocks"].tolist():
        first = block * BLOCK
        page, at = table[row][first // PAGE], first % PAGE
        part = keys[page, at:at + min(BLOCK, used[row] - first)].double()
        bounds[page, :, at // BLOCK, 0] = part.min(dim=0).values
        bounds[page, :, at // BLOCK, 1] = part.max(dim=0).values
    return bounds


def _exact_sparse(state):
    q, keys, values, bounds = state["q"].double(), state["keys"], state["values"], state["bounds"]
    table, used, top = state["table"].long(), state["used"].tolist(), state["case"]["top"]
    rows, heads = q.shape[0], keys.shape[2]
    group = q.shape[1] // heads
    out = torch.zeros_like(q)
    selected = torch.full((rows, heads, top), -1, dtype=torch.int32)
    for row, length in enumerate(used):
        count = -(-length // BLOCK)
        pages = table[row, :-(-length // PAGE)]
        k_all = keys[pages].flatten(0, 1)[:length]
        v_all = values[pages].flatten(0, 1)[:length]
        lo_hi = bounds[pages].double()                                    # [pages, heads, 4, 2, d]
        for h in range(heads):
            query = q[row, h * group:(h + 1) * group]
            lo, hi = (lo_hi[:, h, :, e].flatten(0, 1)[:count] for e in (0, 1))
            best = torch.maximum(query.unsqueeze(1) * lo, query.unsqueeze(1) * hi).sum(-1).max(0).values.tolist()
            kept = set(range(count)) if count <= top else {0, count - 2, count - 1}
            for block in sorted(set(range(count)) - kept, key=lambda b: (-best[b], b))[:max(0, top - len(kept))]:
                kept.add(block)
            kept = sorted(kept)
            selected[row, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            at = torch.cat([torch.arange(b * BLOCK, min(length, (b + 1) * BLOCK)) for b in kept]).to(q.device)
            weight = torch.softmax(query @ k_all[at, h].double().t() / math.sqrt(128), dim=-1)
            out[row, h * group:(h + 1) * group] = weight @ v_all[at, h].double()
    return {"out": out, "selected": selected}


def _exact_controls(state):
    x = state["logits"].double().cpu()
    rows, vocab = x.shape
    history, slots = state["history"].cpu(), state["slots"].tolist()
    lengths, prompts = state["lengths"].tolist(), state["prompts"].tolist()
    r, f, p = (state[name].double().tolist() for name in ("repetition", "frequency", "presence"))
    for row in range(rows):
        told = history[slots[row], :lengths[slots[row]]].long()
        seen = torch.unique(told)
        x[row, seen] = torch.where(x[row, seen] > 0, x[row, seen] / r[row], x[row, seen] * r[row])
        tokens, counts = torch.unique(told[prompts[slots[row]]:], return_counts=True)
        x[row, tokens] -= f[row] * counts.double() + p[row]
    if state["bias"] is not None:
        offsets, tokens, values = (t.cpu() for t in state["bias"])
        for row in range(rows):
            part = slice(int(offsets[row]), int(offsets[row + 1]))
            x[row, tokens[part].long()] += values[part].double()
    if state["mask"] is not None:
        words = state["mask"].cpu()
        for row, mask in enumerate(state["mask_rows"].tolist()):
            if mask >= 0:
                allowed = ((words[mask].unsqueeze(1) >> torch.arange(32, dtype=torch.int32)) & 1).flatten()[:vocab]
                x[row, allowed == 0] = -math.inf
    return x
