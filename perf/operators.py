"""Cases of the paged key/value cache operators: what is called, on which data.

A serving program keeps the keys and values of its sequences in pages of a
fixed number of rows, [pages, kv_heads, page_size, head_dim], and a block
table [batch, columns] that names each sequence's pages in order.  Three
operators work on them (gawee_b200/paged_kv.py):

  append   writes the key and value rows of new tokens into the pages;
  attend   attention of one new token per sequence over its cached keys,
           optionally storing that token's own key and value first, with an
           additive mask, and adding the attention weights that each key
           received to an accumulator;
  evict    keeps the most recent keys and those of the greatest accumulated
           weight, per key/value head, and packs their rows into the first
           rows of the sequence's (or of other) pages.

With `own` false, `run` computes them from elementary torch operations in 32
bits; with `own` true it calls the library.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def _attend(name, batch, heads, kv_heads, dim, page, length, act, cache, ragged=True, mask=False, weights=False,
            new=False):
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "length": length, "act": act, "cache": cache, "ragged": ragged, "mask": mask,
            "weights": weights, "new": new}


def _append(name, batch, kv_heads, dim, page, length, tokens, act, cache):
    return {"name": name, "op": "append", "batch": batch, "kv_heads": kv_heads, "dim": dim, "page": page,
            "length": length, "tokens": tokens, "act": act, "cache": cache}


def _evict(name, batch, kv_heads, dim, page, length, budget, recent, cache, ragged=True):
    return {"name": name, "op": "evict", "batch": batch, "kv_heads": kv_heads, "dim": dim, "page": page,
            "length": length, "budget": budget, "recent": recent, "cache": cache, "ragged": ragged}


def listed():
    return [
        # one token of the 15M decoder (6 heads of 48, fp32) behind a prompt of 256 tokens: the latency of a call
        _attend("attend_f32_6x48_b1", 1, 6, 6, 48, 16, 257, "f32", "f32", new=True),
        # the 135M decoder's heads (9 over 3 of 64, fp32), 64 sequences of up to 2048 tokens
        _attend("attend_f32_9_3x64_b64", 64, 9, 3, 64, 16, 2048, "f32", "f32", new=True),
        # the same heads with a padding mask over a single longer context
        _attend("attend_f32_9_3x64_long_mask", 1, 9, 3, 64, 32, 16385, "f32", "f32", ragged=False, mask=True),
        # a served batch of long contexts in bf16, four query heads to a key/value head: the largest
        _attend("attend_bf16_32_8x128_b32", 32, 32, 8, 128, 16, 8192, "bf16", "bf16"),
        # one very long context: the split along its length
        _attend("attend_bf16_32_8x128_b1", 1, 32, 8, 128, 64, 131071, "bf16", "bf16", ragged=False),
        # odd sizes: 15 heads over 5 of 80, pages of 24 rows, fp32 activations on an fp16 cache, mask and weights
        _attend("attend_f16_15_5x80_odd", 7, 15, 5, 80, 24, 3001, "f32", "f16", mask=True, weights=True),
        # a decode step that also accumulates the weights by which evict chooses
        _attend("attend_f32_9_3x64_weights", 16, 9, 3, 64, 16, 4096, "f32", "f32", weights=True, new=True),
        # one new token of each of 64 sequences
        _append("append_f32_3x64_step", 64, 3, 64, 16, 2048, 1, "f32", "f32"),
        # prompts of up to 1024 tokens, fp32 activations stored in bf16
        _append("append_bf16_8x128_prompts", 24, 8, 128, 16, 4096, 1024, "f32", "bf16"),
        # 16 sequences of the 135M decoder's heads cut to 1024 rows
        _evict("evict_f32_3x64", 16, 3, 64, 16, 2048, 1024, 128, "f32"),
        # a served batch of long contexts cut to a quarter
        _evict("evict_bf16_8x128_b32", 32, 8, 128, 16, 8192, 2048, 256, "bf16"),
        # one very long context
        _evict("evict_bf16_8x128_b1", 1, 8, 128, 64, 65537, 4097, 255, "bf16", ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "evict"])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 6, 8, 12])
    dim = rng.choice([8, 32, 40, 48, 64, 64, 80, 96, 112, 128, 128, 192, 256])
    page = rng.choice([1, 7, 8, 16, 16, 24, 32, 64, 100, 128, 256])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f32"), ("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"),
                             ("f32", "bf16"), ("f32", "f16")])
    # keys of the whole padded batch, so that no drawn case holds more than the largest listed one
    keys = min(1 << 17, (1 << 28) // (SIZES[cache] * kv_heads * dim))
    length = _log(rng, 1, keys)
    batch = _log(rng, 1, max(1, min(256, keys // length)))
    if op == "attend":
        group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
        c = _attend("", batch, kv_heads * group, kv_heads, dim, page, length, act, cache,
                    ragged=rng.random() < 0.7, mask=rng.random() < 0.3, weights=rng.random() < 0.3,
                    new=rng.random() < 0.4)
    elif op == "append":
        c = _append("", batch, kv_heads, dim, page, length, _log(rng, 1, length), act, cache)
    else:
        budget = _log(rng, 1, length)
        c = _evict("", batch, kv_heads, dim, page, length, budget, rng.randint(0, budget), cache,
                   ragged=rng.random() < 0.7)
    del c["name"]
    return c


# --- what a case's shape says ------------------------------------------------

def _lengths(case):
    """Cached keys of each sequence (attend: the new token's among them): up
    to the case's length, one of them exactly that; a property of the case,
    not of the seed, so that the work is."""
    b, n = case["batch"], case["length"]
    if not case.get("ragged", True):
        return [n] * b
    r = random.Random("%d %d %d" % (b, n, case["dim"]))
    got = [r.randint(max(1, n // 8), n) for _ in range(b)]
    if b > 4:
        got[r.randrange(b)] = 1
        if not case.get("new"):
            got[r.randrange(b)] = 0
    got[r.randrange(b)] = n
    return got


def _new_tokens(case):
    """append: (new tokens, rows already cached) of each sequence."""
    lens = _lengths(case)
    r = random.Random("new %d %d" % (case["batch"], case["tokens"]))
    got = []
    for n in lens:
        t = min(n, case["tokens"] if case["tokens"] == 1 else r.randint(max(1, case["tokens"] // 4), case["tokens"]))
        got.append((t, n - t))
    return got


def work(case):
    es, dim, kv = SIZES[case["cache"]], case["dim"], case["kv_heads"]
    row = 2 * kv * dim * es  # a key's and its value's rows over the heads
    lens = _lengths(case)
    if case["op"] == "attend":
        keys = sum(lens)
        ea = SIZES[case["act"]]
        nbytes = keys * row + 2 * case["batch"] * case["heads"] * dim * ea + 4 * case["batch"]
        nbytes += sum(4 * -(-n // case["page"]) for n in lens)
        if case["mask"]:
            nbytes += 4 * keys
        if case["weights"]:
            nbytes += 8 * keys * kv
        if case["new"]:  # read from the call's arguments and stored, in place of being read from the pages
            nbytes += case["batch"] * 2 * kv * dim * ea
        return {"bytes": nbytes, "flops": 4 * keys * case["heads"] * dim}
    if case["op"] == "append":
        t = sum(n for n, _ in _new_tokens(case))
        return {"bytes": t * (2 * kv * dim * SIZES[case["act"]] + row + 8), "flops": 0}
    moved = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": 2 * moved * row + 4 * kv * (sum(lens) + moved) + 4 * case["batch"] * kv * case["budget"],
            "flops": 0}


# --- inputs --------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    b, kv, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    cache = DTYPES[case["cache"]]
    lens = _lengths(case)
    own_pages = [-(-n // page) for n in lens]
    cols = max(own_pages) + 2
    to_pages = [-(-min(n, case["budget"]) // page) for n in lens] if case["op"] == "evict" else [0] * b
    num_pages = sum(own_pages) + sum(to_pages) + 3
    perm = torch.randperm(num_pages, generator=gen, device=dev).to(torch.int32)

    def table(counts, first):
        # unused columns hold -1, as an allocator leaves them
        at = torch.full((b, cols), -1, dtype=torch.int64)
        for i, c in enumerate(counts):
            at[i, :c] = torch.arange(first, first + c)
            first += c
        at = at.to(dev)
        return torch.where(at < 0, at.to(torch.int32), perm[at.clamp(min=0)])

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(scale).to(dtype)

    def pages():
        return torch.randn(num_pages, kv, page, dim, generator=gen, device=dev, dtype=cache)

    s = {"case": case, "k_pages": pages(), "v_pages": pages(), "table": table(own_pages, 0),
         "lengths": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if case["op"] == "attend":
        act = DTYPES[case["act"]]
        s["scale"] = 1.0 / math.sqrt(dim)
        s["q"] = normal(b, case["heads"], dim, dtype=act, scale=2.0)
        s["out"] = torch.empty_like(s["q"])
        s["k"] = normal(b, kv, dim, dtype=act) if case["new"] else None
        s["v"] = normal(b, kv, dim, dtype=act) if case["new"] else None
        s["mask"] = s["weights"] = s["weights_out"] = None
        if case["mask"]:  # padded in front, by up to a quarter of the sequence
            pad = (torch.rand(b, 1, generator=gen, device=dev) * 0.25 * s["lengths"].view(b, 1)).floor()
            at = torch.arange(cols * page, device=dev).view(1, -1)
            s["mask"] = torch.where(at < pad, float("-inf"), 0.0).to(torch.float32)
        if case["weights"]:  # what earlier steps left: heavy-tailed, never negative
            s["weights"] = torch.rand(b, kv, cols * page, generator=gen, device=dev).pow_(8).mul_(4.0)
            s["weights_out"] = torch.zeros_like(s["weights"])
    elif case["op"] == "append":
        act = DTYPES[case["act"]]
        new = _new_tokens(case)
        seq = [i for i, (t, _) in enumerate(new) for _ in range(t)]
        pos = [n + j for t, n in new for j in range(t)]
        s["k"] = normal(len(seq), kv, dim, dtype=act)
        s["v"] = normal(len(seq), kv, dim, dtype=act)
        s["sequences"] = torch.tensor(seq, dtype=torch.int32, device=dev)
        s["positions"] = torch.tensor(pos, dtype=torch.int32, device=dev)
    else:
        s["to_table"] = table(to_pages, sum(own_pages))
        s["weights"] = torch.rand(b, kv, cols * page, generator=gen, device=dev).pow_(8).mul_(4.0)
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["kept"] = torch.empty(b, kv, case["budget"], dtype=torch.int32, device=dev)
        s["lengths_out"] = torch.empty_like(s["lengths"])
    if own:
        from gawee_b200.paged_kv import PagedKV
        s["kv"] = PagedKV(case["cache"], case.get("heads", kv), kv, dim, page, num_pages, max_batch=b, max_pages=cols,
                          weights=bool(case.get("weights")))
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        kv, stream = s["kv"], torch.cuda.current_stream()
        if op == "attend":
            kv.attend(s["k_pages"], s["v_pages"], s["q"], s["table"], s["lengths"], s["out"], scale=s["scale"],
                      k=s["k"], v=s["v"], mask=s["mask"], weights=s["weights"], weights_out=s["weights_out"],
                      stream=stream)
            got = [s["out"]]
            if s["weights"] is not None:
                got.append(s["weights_out"])
            return got + ([s["k_pages"], s["v_pages"]] if s["k"] is not None else [])
        if op == "append":
            kv.append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["table"], s["positions"],
                      sequences=s["sequences"], stream=stream)
            return [s["k_pages"], s["v_pages"]]
        kv.evict(s["k_pages"], s["v_pages"], s["weights"], s["table"], s["lengths"], s["case"]["budget"],
                 s["case"]["recent"], s["kept"], s["weights_out"], s["lengths_out"], to_table=s["to_table"],
                 stream=stream)
        return [s["k_pages"], s["v_pages"], s["kept"], s["weights_out"], s["lengths_out"]]
    return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict}[op](s)


# --- the plain forms ---------------------------------------------------------------

def _store(pages, rows, page_ids, slots):
    pages[page_ids, :, slots] = rows.to(pages.dtype)


def _plain_append(s):
    page = s["case"]["page"]
    pos, seq = s["positions"].long(), s["sequences"].long()
    ids = s["table"][seq, pos // page].long()
    _store(s["k_pages"], s["k"], ids, pos % page)
    _store(s["v_pages"], s["v"], ids, pos % page)
    return [s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    case = s["case"]
    b, h, kv, dim, page = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "page"))
    lens = s["lengths"].long()
    if s["k"] is not None:
        last = lens - 1
        ids = s["table"].gather(1, (last // page).view(b, 1)).view(b).long()
        _store(s["k_pages"], s["k"], ids, last % page)
        _store(s["v_pages"], s["v"], ids, last % page)
    ids = s["table"].clamp(min=0).long()
    n = ids.shape[1] * page
    valid = (torch.arange(n, device=ids.device).view(1, n) < lens.view(b, 1)).view(b, 1, 1, n)
    k = s["k_pages"][ids].float().permute(0, 2, 1, 3, 4).reshape(b, kv, n, dim)
    score = torch.matmul(s["q"].float().view(b, kv, h // kv, dim), k.transpose(2, 3)) * s["scale"]
    del k
    if s["mask"] is not None:
        score = score + s["mask"].view(b, 1, 1, n)
    score = score.masked_fill(~valid, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = s["v_pages"][ids].float().permute(0, 2, 1, 3, 4).reshape(b, kv, n, dim)
    v = v.masked_fill(~valid.view(b, 1, n, 1), 0.0)
    out = torch.matmul(p, v).view(b, h, dim).to(s["q"].dtype)
    got = [out]
    if s["weights"] is not None:
        got.append(torch.where(valid.view(b, 1, n), s["weights"] + p.sum(2), s["weights_out"]))
    return got + ([s["k_pages"], s["v_pages"]] if s["k"] is not None else [])


def _plain_evict(s):
    case = s["case"]
    b, kv, page, budget = case["batch"], case["kv_heads"], case["page"], case["budget"]
    w, lens = s["weights"], s["lengths"].long().view(b, 1, 1)
    n = w.shape[2]
    at = torch.arange(n, device=w.device).view(1, 1, n)
    key = torch.where(at >= lens - case["recent"], float("inf"), w)
    key = torch.where(at >= lens, float("-inf"), key)
    if n < budget:  # a budget beyond the table's rows: nothing is evicted
        key = torch.nn.functional.pad(key, (0, budget - n), value=float("-inf"))
    # equal weights: the lowest position first
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    slot = torch.arange(budget, device=w.device).view(1, 1, budget)
    new = torch.minimum(lens, torch.full_like(lens, budget))
    kept = torch.where(slot < new, torch.where(lens <= budget, slot, order), -1)
    bi, hi, si = (slot < new).expand(b, kv, budget).nonzero(as_tuple=True)
    src = kept[bi, hi, si]
    weights = torch.zeros_like(w)
    weights[bi, hi, si] = w[bi, hi, src]
    from_page, to_page = s["table"][bi, src // page].long(), s["to_table"][bi, si // page].long()
    for pages in (s["k_pages"], s["v_pages"]):
        pages[to_page, hi, si % page] = pages[from_page, hi, src % page]
    weights = torch.where(at < lens, weights, s["weights_out"])  # rows behind the sequence stay
    return [s["k_pages"], s["v_pages"], kept.to(torch.int32), weights, new.view(b).to(torch.int32)]


# --- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    table, lens = s["table"].cpu().tolist(), s["lengths"].cpu().tolist()

    def rows(pages, i, count):
        """The first `count` rows of sequence i: [kv, count, dim]."""
        ids = torch.tensor(table[i][:-(-count // page)], dtype=torch.long, device=pages.device)
        return pages.index_select(0, ids).transpose(0, 1).flatten(1, 2)[:, :count]

    def put(pages, which, values):
        """Row `which[j]` = (page, row) takes values[j], [tokens, kv, dim]."""
        flat = pages.transpose(1, 2).contiguous().view(-1, kv, dim)
        at = torch.tensor([p * page + r for p, r in which], dtype=torch.long, device=pages.device)
        flat.index_copy_(0, at, values.to(pages.dtype))
        return flat.view(-1, page, kv, dim).transpose(1, 2).contiguous()

    if case["op"] == "append":
        which = [(table[i][p // page], p % page)
                 for i, p in zip(s["sequences"].cpu().tolist(), s["positions"].cpu().tolist())]
        return [put(s["k_pages"], which, s["k"]), put(s["v_pages"], which, s["v"])]
    if case["op"] == "attend":
        k_pages, v_pages = s["k_pages"], s["v_pages"]
        if case["new"]:
            which = [(table[i][(n - 1) // page], (n - 1) % page) for i, n in enumerate(lens)]
            k_pages, v_pages = put(k_pages, which, s["k"]), put(v_pages, which, s["v"])
        group = case["heads"] // kv
        out = torch.zeros(case["batch"], case["heads"], dim, dtype=torch.float64, device=k_pages.device)
        acc = None if s["weights"] is None else s["weights_out"].double()
        for i, n in enumerate(lens):
            for j in range(kv if n else 0):
                kk, vv = rows(k_pages, i, n)[j].double(), rows(v_pages, i, n)[j].double()
                x = torch.einsum("gd,nd->gn", s["q"][i, j * group:(j + 1) * group].double(), kk) * s["scale"]
                if s["mask"] is not None:
                    x = x + s["mask"][i, :n].double()
                p = torch.softmax(x, dim=1)
                out[i, j * group:(j + 1) * group] = torch.einsum("gn,nd->gd", p, vv)
                if acc is not None:
                    acc[i, j, :n] = s["weights"][i, j, :n].double() + p.sum(0)
        return [out] + ([] if acc is None else [acc]) + ([k_pages, v_pages] if case["new"] else [])
    budget, recent = case["budget"], case["recent"]
    to = s["to_table"].cpu().tolist()
    kept = torch.full((case["batch"], kv, budget), -1, dtype=torch.int64)
    w = s["weights"].cpu().double()
    w_out = s["weights_out"].cpu().double()
    k_pages, v_pages = s["k_pages"].clone(), s["v_pages"].clone()
    for i, n in enumerate(lens):
        m = min(n, budget)
        w_out[i, :, :n] = 0
        for j in range(kv if n else 0):
            keep = list(range(n))
            if n > budget:
                old = torch.sort(-w[i, j, :n - recent], stable=True).indices[:budget - recent].tolist()
                keep = sorted(old) + list(range(n - recent, n))
            kept[i, j, :m] = torch.tensor(keep)
            w_out[i, j, :m] = w[i, j, keep]
            at = torch.tensor(keep, device=k_pages.device)
            for pages, into in ((s["k_pages"], k_pages), (s["v_pages"], v_pages)):
                moved = rows(pages, i, n)[j].index_select(0, at)
                for c in range(-(-m // page)):
                    part = moved[c * page:(c + 1) * page]
                    into[to[i][c], j, :part.shape[0]] = part
    return [k_pages, v_pages, kept.to(torch.int32), w_out, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32)]
