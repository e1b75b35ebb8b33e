"""Operators that a serving loop calls around the linears, as cases that can be timed and checked: new keys and values into
the pages of a cache, attention of prompts and of single tokens over those pages, logits to probabilities, and drafted tokens
against them.

A case is a dict of plain values.  `prepare` makes what a program holds before the call, `run` is one pass through an
operator (with `own` the framework's, else its plain form), `exact` the same outputs in 64 bits, `work` the bytes and
operations that a pass cannot do without."""
import math
import os
import sys

import numpy as np
import torch

own = False

# heads, key heads, head size of the decoders this repository describes
HEADS = {"896": (14, 2, 64), "1536": (12, 2, 128), "2048": (16, 4, 128)}
VOCABS = (32000, 151936)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NEAR = 128  # distances with a bias of their own


def listed():
    return [
        # one user in the middle of an answer: the smallest call, latency
        dict(name="decode_chat", kind="decode", model="896", dtype="bf16", seqs=1, tokens=1, length=93, spread=0, page=16, window=0, keep=0, rel=False),
        # many users at once, contexts of all lengths
        dict(name="decode_batch", kind="decode", model="1536", dtype="bf16", seqs=64, tokens=1, length=1100, spread=900, page=64, window=0, keep=0, rel=False),
        # long conversations, the tokens of a draft checked together
        dict(name="decode_drafts", kind="decode", model="2048", dtype="fp16", seqs=32, tokens=5, length=12000, spread=4000, page=32, window=0, keep=0, rel=False),
        # a short question
        dict(name="prompt_chat", kind="prompt", model="896", dtype="bf16", counts="41", before="0", page=16, window=0, keep=0, rel=False),
        # portions of several prompts in one step, window and first tokens
        dict(name="prompt_portions", kind="prompt", model="1536", dtype="bf16", counts="700 1 512 333 1025", before="0 2311 1536 77 0", page=64,
             window=512, keep=4, rel=False),
        # a long document in one step
        dict(name="prompt_document", kind="prompt", model="2048", dtype="bf16", counts="8192", before="0", page=128, window=0, keep=0, rel=False),
        # a token of every sequence of a batch
        dict(name="append_token", kind="append", model="1536", dtype="bf16", counts="1 " * 64, before="11 37 500 1023 64 63 65 2 " * 8, page=64),
        # a step of prompts
        dict(name="append_prompts", kind="append", model="2048", dtype="fp16", counts="1900 1500 77 2048 1311 640 1999 1",
             before="0 311 0 0 1024 16 0 5", page=32),
        # one sequence's draft
        dict(name="verify_one", kind="verify", seqs=1, drafts=4, vocab=32000),
        # drafts of a batch
        dict(name="verify_batch", kind="verify", seqs=64, drafts=5, vocab=151936),
        # logits of one sequence's draft
        dict(name="probs_one", kind="probs", rows=5, vocab=32000, temperature=0.8),
        # logits of a batch of drafts
        dict(name="probs_batch", kind="probs", rows=384, vocab=151936, temperature=1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "decode", "prompt", "prompt", "prompt", "append", "verify", "probs"))
    if kind == "verify":
        return dict(kind=kind, seqs=_log(rng, 1, 64), drafts=rng.randint(1, 8), vocab=rng.choice(VOCABS))
    if kind == "probs":
        return dict(kind=kind, rows=_log(rng, 1, 384), vocab=rng.choice(VOCABS), temperature=rng.choice((0.0, 0.6, 1.0, 1.3)))
    case = dict(kind=kind, model=rng.choice(sorted(HEADS)), dtype=rng.choice(("bf16", "bf16", "fp16")), page=rng.choice((16, 32, 64, 128, 256, 48)))
    windowed = rng.random() < 0.4
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        length = _log(rng, 8, 300000 // seqs)
        case.update(seqs=seqs, tokens=rng.choice((1, 1, 1, 2, 4, 5, 8)), length=length, spread=int(length * rng.choice((0.0, 0.3, 0.8))))
        case["length"] = max(case["length"], case["spread"] + case["tokens"])
    else:
        seqs, rows = _log(rng, 1, 8), _log(rng, 2, 7000)
        counts = [_log(rng, max(1, rows // seqs // 8), max(1, rows // seqs)) for _ in range(seqs)]
        case.update(counts=" ".join(map(str, counts)), before=" ".join(str(rng.choice((0, 0, _log(rng, 1, 4000)))) for _ in counts))
    if kind != "append":
        case.update(window=_log(rng, 64, 4096) if windowed else 0, keep=rng.choice((0, 1, 4, 17)) if windowed else 0, rel=rng.random() < 0.25)
    return case


# ------------------------------------------------------------------------------------------------ inputs from a seed
def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + what)


def _ints(text):
    return [int(x) for x in text.split()]


def _lengths(case, seed):
    """(tokens that every sequence brings, tokens it has with them)."""
    if "counts" in case:
        counts = _ints(case["counts"])
        return counts, [c + b for c, b in zip(counts, _ints(case["before"]))]
    rng = np.random.default_rng(seed)
    n = [int(case["length"] - rng.integers(0, case["spread"] + 1)) for _ in range(case["seqs"])]
    return [case["tokens"]] * case["seqs"], n


def _table(lengths, page, seed):
    """Pages in an order of their own, as a cache in use has them; a few that belong to nobody among them."""
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 3
    order = np.random.default_rng(seed + 7).permutation(pages)
    table, at = np.zeros((len(lengths), max(need)), np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return pages, table


def _randn(shape, dtype, gen):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(generator=gen)


def _inputs(case, seed):
    """Tensors of a case by name."""
    kind = case["kind"]
    if kind == "probs":
        return dict(logits=_randn((case["rows"], case["vocab"]), torch.float32, _gen(seed, 1)).mul_(2.5))
    if kind == "verify":
        s, k, v = case["seqs"], case["drafts"], case["vocab"]
        z = _randn((s, k + 1, v), torch.float32, _gen(seed, 1)).mul_(2.5)
        noise = _randn((s, k, v), torch.float32, _gen(seed, 2))
        draft = torch.softmax(z[:, :k] + 0.4 * noise, dim=-1)
        del noise
        target = torch.softmax(z, dim=-1)
        # drafted tokens as the draft model would sample them
        c = torch.cumsum(draft.double(), dim=-1)
        at = torch.rand((s, k, 1), dtype=torch.float64, device="cuda", generator=_gen(seed, 3)) * c[..., -1:]
        tokens = torch.searchsorted(c, at, right=True).clamp_(max=v - 1)[..., 0].to(torch.int32)
        del c
        return dict(target=target, draft=draft, tokens=tokens, accept=torch.rand((s, k), device="cuda", generator=_gen(seed, 4)),
                    pick=torch.rand((s,), device="cuda", generator=_gen(seed, 5)))
    heads, kv, dim = HEADS[case["model"]]
    dtype = DTYPES[case["dtype"]]
    counts, lengths = _lengths(case, seed)
    pages, table = _table(lengths, case["page"], seed)
    rows = sum(counts)
    out = dict(k=_randn((pages, kv, case["page"], dim), dtype, _gen(seed, 1)), v=_randn((pages, kv, case["page"], dim), dtype, _gen(seed, 2)),
               table=torch.from_numpy(table).cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
               q_start=torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda"))
    if kind == "append":
        out.update(new_k=_randn((rows, kv, dim), dtype, _gen(seed, 3)), new_v=_randn((rows, kv, dim), dtype, _gen(seed, 4)))
    else:
        out.update(q=_randn((rows, heads, dim), dtype, _gen(seed, 3)), sink=None, bias=None)
        if case["rel"]:
            out.update(sink=_randn((heads,), torch.float32, _gen(seed, 4)), bias=_randn((heads, NEAR + 1), torch.float32, _gen(seed, 5)))
    return out


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if "k" in state:
        counts, lengths = _lengths(case, seed)
        state.update(most=max(counts), longest=max(lengths))  # what the program knows on the host
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        sys.path[:0] = [p for p in [os.path.join(os.getcwd(), "mllm-advanced_b200")] if p not in sys.path]
        from mllm_b200 import drafts, paged
        return _own(case, state, drafts, paged)
    return {"decode": _attention, "prompt": _attention, "append": _append, "verify": _verify, "probs": _probs}[case["kind"]](case, state)


def _own(case, t, drafts, paged):
    kind = case["kind"]
    if kind == "probs":
        return drafts.probabilities(t["logits"], case["temperature"])
    if kind == "verify":
        return drafts.verify(t["target"], t["draft"], t["tokens"], t["accept"], t["pick"])
    if kind == "append":
        paged.append(t["k"], t["v"], t["new_k"], t["new_v"], t["table"], t["lengths"], t["q_start"])
        return t["k"], t["v"]
    look = dict(window=case["window"], keep=case["keep"], sink=t["sink"], bias=t["bias"])
    if kind == "decode":
        return paged.decode_attention(t["q"], t["k"], t["v"], t["table"], t["lengths"], **look)
    return paged.prompt_attention(t["q"], t["k"], t["v"], t["table"], t["lengths"], t["q_start"], **look)


def _contexts(pool, table, longest):
    """Every sequence's rows, [sequences, kv heads, longest, dim] in 32 bits."""
    page = pool.shape[2]
    rows = pool[table[:, :(longest + page - 1) // page].long()]  # [sequences, pages, kv heads, page, dim]
    return rows.transpose(1, 2).flatten(2, 3)[:, :, :longest].float()


def _attention(case, t):
    heads, kv, dim = HEADS[case["model"]]
    group, window, keep, most, longest = heads // kv, case["window"], case["keep"], t["most"], t["longest"]
    k, v = _contexts(t["k"], t["table"], longest), _contexts(t["v"], t["table"], longest)
    seqs, count = k.shape[0], t["q_start"][1:] - t["q_start"][:-1]
    place = torch.arange(most, device="cuda")
    row = (t["q_start"][:-1, None] + place).clamp_(max=t["q"].shape[0] - 1)  # [sequences, most]: rows behind a sequence's own are computed, not kept
    q = t["q"][row.long()].float().reshape(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4)
    i = ((t["lengths"] - count)[:, None] + place)[:, :, None]
    j = torch.arange(longest, device="cuda")
    hidden = j > i
    if window:
        hidden = hidden | ((j <= i - window) & (j >= keep))
    hidden = hidden[:, None, None]
    z = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).mul_(dim ** -0.5).reshape(seqs, kv, group, most, longest)
    if t["bias"] is not None:
        z += t["bias"][:, (i - j).clamp_(0, NEAR).long()].reshape(kv, group, seqs, most, longest).permute(2, 0, 1, 3, 4)
    z.masked_fill_(hidden, float("-inf"))
    m = z.max(dim=-1, keepdim=True).values
    if t["sink"] is not None:
        sink = t["sink"].reshape(1, kv, group, 1, 1)
        m = torch.maximum(m, sink)
    w = z.sub_(m).exp_()
    total = w.sum(dim=-1, keepdim=True)
    if t["sink"] is not None:
        total = total + torch.exp(sink - m)
    v = v.masked_fill_((j >= t["lengths"][:, None])[:, None, :, None], 0.0)
    o = (torch.matmul(w.flatten(2, 3), v).reshape(seqs, kv, group, most, dim) / total).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    return o[place < count[:, None]].to(t["q"].dtype)


def _append(case, t):
    page = case["page"]
    row = torch.arange(t["new_k"].shape[0], device="cuda", dtype=torch.int32)
    s = torch.searchsorted(t["q_start"], row, right=True) - 1
    pos = (t["lengths"][s] + row - t["q_start"][s + 1]).long()
    at, inside = t["table"][s, pos // page].long(), pos % page
    t["k"][at, :, inside] = t["new_k"]
    t["v"][at, :, inside] = t["new_v"]
    return t["k"], t["v"]


def _verify(case, t):
    k, v = case["drafts"], case["vocab"]
    tokens = t["tokens"].long()
    p = t["target"][:, :k].gather(2, tokens[..., None])[..., 0].double()
    q = t["draft"].gather(2, tokens[..., None])[..., 0].double()
    good = t["accept"].double() * q < p
    accepted = good.long().cumprod(dim=1).sum(dim=1)
    s = torch.arange(case["seqs"], device="cuda")
    left = t["target"][s, accepted].double()
    refused = accepted < k
    rest = (left - t["draft"][s, accepted.clamp(max=k - 1)].double()).clamp_(min=0)
    mass = torch.where((refused & (rest.sum(dim=1) > 0))[:, None], rest, left)
    c = torch.cumsum(mass, dim=1)
    after = c > t["pick"].double()[:, None] * c[:, -1:]
    index = torch.arange(v, device="cuda")
    nxt = torch.where(after, index, v).min(dim=1).values
    last = torch.where(mass > 0, index, -1).max(dim=1).values
    nxt = torch.where(nxt < v, nxt, last)
    place = torch.arange(k + 1, device="cuda")
    out = torch.where(place < accepted[:, None], torch.nn.functional.pad(tokens, (0, 1)), torch.full_like(place, -1))
    out = torch.where(place == accepted[:, None], nxt[:, None], out)
    return accepted.to(torch.int32), out.to(torch.int32)


def _probs(case, t):
    z = t["logits"]
    if case["temperature"] == 0:
        top = z.max(dim=1, keepdim=True).values
        index = torch.arange(z.shape[1], device="cuda")
        first = torch.where(z == top, index, z.shape[1]).min(dim=1, keepdim=True).values
        return (index == first).float()
    w = torch.exp((z - z.max(dim=1, keepdim=True).values) / case["temperature"])
    return w / w.sum(dim=1, keepdim=True)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """Written apart from the plain forms: attention per query row block with an additive mask over the whole context, the
    inverse distribution function through a search."""
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "verify":
        return None  # whole numbers, which the plain form computes in 64 bits
    if kind == "probs":
        z = t["logits"].double()
        if case["temperature"] == 0:
            return torch.zeros_like(z).scatter_(1, z.argmax(dim=1, keepdim=True), 1.0)
        z = z / case["temperature"]
        return torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    heads, kv, dim = HEADS[case["model"]]
    counts, lengths = _lengths(case, seed)
    table, page = t["table"].cpu().long() if kind == "append" else t["table"].long(), case["page"]
    if kind == "append":
        pools, row = [t["k"].double(), t["v"].double()], 0
        for s, (count, n) in enumerate(zip(counts, lengths)):
            for c in range(count):
                at, inside = int(table[s, (n - count + c) // page]), (n - count + c) % page
                for pool, new in zip(pools, (t["new_k"], t["new_v"])):
                    pool[at, :, inside] = new[row + c].double()
            row += count
        return tuple(pools)
    out, row = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda"), 0
    for s, (count, n) in enumerate(zip(counts, lengths)):
        place = torch.arange(n, device="cuda")
        ids, inside = table[s, place // page], place % page
        for r0 in range(0, count, 512):
            r1 = min(count, r0 + 512)
            pos = n - count + torch.arange(r0, r1, device="cuda")
            dist = pos[:, None] - place[None, :]
            seen = dist >= 0
            if case["window"]:
                seen &= (dist < case["window"]) | (place < case["keep"])[None, :]
            some = seen.any(dim=0)
            for h in range(heads):
                g = h // (heads // kv)
                keys, values = t["k"][ids[some], g, inside[some]].double(), t["v"][ids[some], g, inside[some]].double()
                z = t["q"][row + r0:row + r1, h].double() @ keys.T / math.sqrt(dim)
                if t["bias"] is not None:
                    z = z + t["bias"][h].double()[dist[:, some].clamp(0, NEAR)]
                z = torch.where(seen[:, some], z, torch.full_like(z, -math.inf))
                if t["sink"] is not None:
                    z = torch.cat([z, t["sink"][h].double().expand(r1 - r0, 1)], dim=1)
                    values = torch.cat([values, values.new_zeros(1, dim)])
                out[row + r0:row + r1, h] = torch.softmax(z, dim=1) @ values
        row += count
    return out


# ------------------------------------------------------------------------------------------------ what a pass needs
def _visible(case, count, n):
    """(pairs of a query and a key it sees, keys that some query sees)."""
    w, keep = case["window"], case["keep"]
    i = np.arange(n - count, n, dtype=np.int64)
    if not w:
        return int((i + 1).sum()), n
    lo = np.maximum(0, i - w + 1)
    pairs = int((i + 1 - lo + np.minimum(keep, lo)).sum())
    first = int(lo[0])
    return pairs, n - first + min(keep, first)


def work(case):
    kind = case["kind"]
    if kind == "probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 8 * n, "flops": 4 * n}
    if kind == "verify":
        s, k, v = case["seqs"], case["drafts"], case["vocab"]
        # the rows of the first refused place, and what decides on the drafted tokens
        return {"bytes": s * (2 * v * 4 + k * 16 + 4 + (k + 2) * 4), "flops": 3 * s * v}
    heads, kv, dim = HEADS[case["model"]]
    if kind == "append":
        n = sum(_ints(case["counts"])) * kv * dim * 2
        return {"bytes": 2 * n * 2, "flops": 0}
    seqs = zip(*_lengths(case, 0)) if "counts" in case else [(case["tokens"], case["length"] - case["spread"] // 2)] * case["seqs"]
    pairs = keys = rows = 0
    for count, n in seqs:
        a, b = _visible(case, count, n)
        pairs, keys, rows = pairs + a, keys + b, rows + count
    return {"bytes": keys * kv * dim * 2 * 2 + rows * heads * dim * 2 * 2, "flops": 4 * dim * heads * pairs}
