"""Cases, inputs and plain forms of the serving operators: attention over packed prompts, attention of one new
token over a paged key-value cache, and the write of new keys and values into that cache.

`run` computes an operator in elementary torch operations in 32 bits, rounded once at the end, or, where `own`
is set, makes the calls that a user of this package makes.  `exact` is the operator's definition in 64 bits."""
import importlib
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
#: most work of a drawn case: visible query-key pairs x heads x head dim, scores of the padded batch, cache bytes
MOST_PAIRS = 32 * 128 * 16384 * 16385 // 2
MOST_SCORES = 32 * 16384 * 16384
MOST_CACHE = 32 * 8 * 128 * 16384 * 4


def listed():
    return [
        # a short question to a small model: latency is all that counts
        {"name": "prompt_short", "op": "prompt", "type": "bf16", "heads": 8, "kv_heads": 2, "dim": 64,
         "q_lens": "33", "k_lens": "33", "fused": True},
        # a batch of ordinary requests, packed, with grouped heads; one slot of the batch is empty
        {"name": "prompt_ragged", "op": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "q_lens": "513,1,1999,0,128,67,2048,300,1021,5,777,1400,250", "k_lens": "same", "fused": True},
        # the GPT-3 head shape of this repository's benchmark (96 heads of 128, 4 sequences of 1024), causal
        {"name": "prompt_gpt3_1k", "op": "prompt", "type": "fp16", "heads": 96, "kv_heads": 96, "dim": 128,
         "q_lens": "1024,1024,1024,1024", "k_lens": "same", "fused": True},
        # later pieces of prompts that are worked off in pieces: the keys reach back before the first query
        {"name": "prompt_piece_d64", "op": "prompt", "type": "fp16", "heads": 16, "kv_heads": 16, "dim": 64,
         "q_lens": "512,384,77", "k_lens": "4096,1400,2125", "fused": False},
        # one long document
        {"name": "prompt_long", "op": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "q_lens": "16384", "k_lens": "same", "fused": True},
        # one user's chat, the smallest decoding call
        {"name": "decode_one", "op": "decode", "type": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "1023", "page": 16, "order": "heads", "lse": False},
        # a full serving batch, contexts of every length, one slot of the batch idle
        {"name": "decode_batch", "op": "decode", "type": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "lens": "8192,17,4097,1,2500,0,6000,333,1024,7777,50,3500,900,129,5111,2049,64,1800,4444,700,15,"
                             "8000,256,1200,3333,600,95,5800,2222,48,1500,6500", "page": 64, "order": "heads",
         "lse": False},
        # one very long context; the partial statistics are wanted for a merge with another part
        {"name": "decode_long", "op": "decode", "type": "fp16", "cache": "fp16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "130001", "page": 16, "order": "tokens", "lse": True},
        # the benchmark's 96 heads without grouping: one query row for every key-value head
        {"name": "decode_gpt3_2k", "op": "decode", "type": "fp16", "cache": "fp16", "heads": 96, "kv_heads": 96,
         "dim": 128, "lens": "2048,2047,1900,2000,1024,1500,2048,1777", "page": 32, "order": "heads", "lse": False},
        # a cache of 8-bit values with a scale for each head
        {"name": "decode_e4m3", "op": "decode", "type": "bf16", "cache": "e4m3", "heads": 64, "kv_heads": 8, "dim": 128,
         "lens": "16384,9000,16001,12345,16384,7000,15000,11111,16384,10000,13000,14000,16384,8000,12000,9999",
         "page": 128, "order": "heads", "lse": False},
        # a packed batch of prompts enters the cache
        {"name": "append_prompts", "op": "append", "type": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "new": "513,1,1999,0,128,67,2048,300,1021,5,777,1400,250", "before": "0,900,0,40,0,31,0,0,17,0,0,0,0",
         "page": 64, "order": "heads"},
        # one token of every sequence of a decoding batch enters an 8-bit cache
        {"name": "append_step_e4m3", "op": "append", "type": "bf16", "cache": "e4m3", "heads": 64, "kv_heads": 8,
         "dim": 128, "new": "1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1", "before": "900,17,409,0,250,63,600,333,102,777,50,350,90,12,511,204",
         "page": 128, "order": "heads"},
    ]


def log_size(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def text(lens):
    return ",".join(str(n) for n in lens)


def numbers(lens):
    return [int(n) for n in lens.split(",")]


def draw(rng):
    op = rng.choice(("prompt", "prompt", "decode", "decode", "append"))
    dim = rng.choice((64, 128, 128, 128, 32, 40, 72, 80, 96, 112, 120))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 16, 32, 40, 96))
    heads = kv_heads * rng.choice([g for g in (1, 1, 2, 3, 4, 5, 7, 8, 16, 24) if kv_heads * g <= 96])
    kind = rng.choice(("fp16", "bf16"))
    if op == "prompt":
        many, top = log_size(rng, 1, 24), log_size(rng, 2, 16384)
        q_lens = [log_size(rng, 1, top) for _ in range(many)]
        before = [0] * many if rng.random() < 0.6 else [log_size(rng, 1, top) for _ in range(many)]
        while (sum(a * (a + 2 * b) for a, b in zip(q_lens, before)) * heads * dim > 2 * MOST_PAIRS
               or len(q_lens) * heads * max(q_lens) * max(a + b for a, b in zip(q_lens, before)) > MOST_SCORES):
            q_lens, before = [max(1, a // 2 + a % 2) for a in q_lens], [b // 2 for b in before]
            if len(q_lens) > 4:
                q_lens, before = q_lens[:-2], before[:-2]
        k_lens = text(a + b for a, b in zip(q_lens, before)) if any(before) else "same"
        return {"op": op, "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "q_lens": text(q_lens),
                "k_lens": k_lens, "fused": k_lens == "same" and rng.random() < 0.7}
    cache = rng.choice((kind, kind, "e4m3"))
    page, order = rng.choice((16, 16, 32, 64, 128, 256)), rng.choice(("heads", "heads", "tokens"))
    if op == "decode":
        many, top = log_size(rng, 1, 128), log_size(rng, 16, 131072)
        lens = [log_size(rng, 1, top) for _ in range(many)]
        if many > 3 and rng.random() < 0.3:
            lens[rng.randrange(many)] = 0
        while len(lens) * max(lens) * kv_heads * dim * 4 > MOST_CACHE:
            lens = [n // 2 + n % 2 for n in lens] if len(lens) < 4 else lens[: len(lens) * 3 // 4]
        return {"op": op, "type": kind, "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "lens": text(lens), "page": page, "order": order, "lse": rng.random() < 0.4}
    many = log_size(rng, 1, 64)
    new = [1] * many if rng.random() < 0.4 else [log_size(rng, 1, 2048) for _ in range(many)]
    before = [0 if rng.random() < 0.5 else log_size(rng, 1, 1024) for _ in range(many)]
    while sum(new) + sum(before) > 16384 or sum(new) * kv_heads > 65536:
        new, before = [n // 2 + n % 2 for n in new], [n // 2 for n in before]
    return {"op": op, "type": kind, "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim, "new": text(new),
            "before": text(before), "page": page, "order": order}


# ---- inputs -------------------------------------------------------------------------------------------
def k_lens_of(case):
    return numbers(case["q_lens"] if case["k_lens"] == "same" else case["k_lens"])


def offsets(lens):
    total = [0]
    total.extend(sum(lens[: i + 1]) for i in range(len(lens)))
    return torch.tensor(total, dtype=torch.int32, device=DEVICE)


def activations(gen, rows, heads, dim, kind, uneven):
    """Projected activations: about unit variance; keys (`uneven`) carry a few strong channels, as trained models' do."""
    x = torch.randn((rows, heads, dim), generator=gen, device=DEVICE)
    if uneven:
        x = x * torch.exp(0.4 * torch.randn((1, heads, dim), generator=gen, device=DEVICE))
    return x.to(TYPES[kind])


def paged(case, lens, gen):
    """Page table of sequences of these lengths over a shuffled pool with a few spare pages; entries behind a
    sequence's last page are -1."""
    need = torch.tensor([-(-n // case["page"]) for n in lens], device=DEVICE)
    width = max(1, int(need.max()))
    total = int(need.sum()) + 3
    column = torch.arange(width, device=DEVICE)
    index = (need.cumsum(0) - need)[:, None] + column
    table = torch.randperm(total, generator=gen, device=DEVICE)[index.clamp(max=total - 1)]
    return torch.where(column < need[:, None], table, -1).to(torch.int32), total


def cache_of(case, pages, gen):
    """A cache [pages, kv_heads, page, dim] in use: every entry holds something.  Its memory runs over a page's
    heads first or over its tokens first."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["order"] == "tokens":
        shape = (shape[0], shape[2], shape[1], shape[3])
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float16)
    x = (x * 40).to(TYPES["e4m3"]) if case["cache"] == "e4m3" else x.to(TYPES[case["cache"]])
    return x.transpose(1, 2) if case["order"] == "tokens" else x


def scales(case, gen):
    """What one step of an 8-bit cache stands for, for each head; none for a 16-bit cache."""
    if case["cache"] != "e4m3":
        return None, None
    one = torch.rand((2, case["kv_heads"]), generator=gen, device=DEVICE) * 0.02 + 0.015
    return one[0].contiguous(), one[1].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "prompt":
        q_lens, k_lens = numbers(case["q_lens"]), k_lens_of(case)
        s["cu_q"], s["cu_k"] = offsets(q_lens), offsets(k_lens)
        if case["fused"]:  # one projection's output, cut into queries, keys and values
            x = torch.cat([activations(gen, sum(q_lens), n, d, case["type"], n == hk) for n in (h, hk, hk)], 1)
            s["q"], s["k"], s["v"] = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
        else:
            s["q"] = activations(gen, sum(q_lens), h, d, case["type"], False)
            s["k"] = activations(gen, sum(k_lens), hk, d, case["type"], True)
            s["v"] = activations(gen, sum(k_lens), hk, d, case["type"], False)
        return s
    if case["op"] == "decode":
        lens = numbers(case["lens"])
        s["q"] = activations(gen, len(lens), h, d, case["type"], False)
    else:
        new, before = numbers(case["new"]), numbers(case["before"])
        lens = [a + b for a, b in zip(new, before)]
        x = torch.cat([activations(gen, sum(new), n, d, case["type"], False) for n in (h, hk, hk)], 1)
        s["k"], s["v"], s["cu"] = x[:, h:h + hk], x[:, h + hk:], offsets(new)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    s["table"], pages = paged(case, lens, gen)
    s["k_cache"], s["v_cache"] = cache_of(case, pages, gen), cache_of(case, pages, gen)
    s["k_scale"], s["v_scale"] = scales(case, gen)
    return s


# ---- one pass -----------------------------------------------------------------------------------------
def run(s):
    return {"prompt": run_prompt, "decode": run_decode, "append": run_append}[s["case"]["op"]](s)


def package():
    return importlib.import_module("flash-attention_amd")


def softmax_times(scores, visible, v):
    """softmax over the visible keys, times v; zeros and minus infinity where nothing is visible.  [.., q, k], [.., k, d]"""
    scores = scores.masked_fill_(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out, (total.log() + top).squeeze(-1)


def run_prompt(s):
    case = s["case"]
    if own:
        return package().forward_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=True, sync=False)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    lq, lk, many = max(1, max(numbers(case["q_lens"]))), max(1, max(k_lens_of(case))), len(numbers(case["q_lens"]))
    i, j = torch.arange(lq, device=DEVICE), torch.arange(lk, device=DEVICE)
    nq, nk = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None, None], (s["cu_k"][1:] - s["cu_k"][:-1])[:, None, None]
    at_q = (s["cu_q"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    at_k = (s["cu_k"][:-1, None] + j).clamp(max=s["k"].shape[0] - 1).long()
    q = s["q"][at_q].float().permute(0, 2, 1, 3).reshape(many, hk, h // hk * lq, d)
    k = s["k"][at_k].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][at_k].float().permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q * d ** -0.5, k).view(many, hk, h // hk, lq, lk)
    visible = (j <= i[:, None] + (nk - nq)) & (j < nk)  # the last query sees the last key
    out, _ = softmax_times(scores, visible[:, None, None], v[:, :, None])
    out = out.view(many, h, lq, d).transpose(1, 2)
    return out[i < nq[:, :, 0]].to(s["q"].dtype)


def gathered(cache, table, scale):
    """[sequences, kv_heads, table's positions, dim] in 32 bits."""
    pages = table.clamp(min=0).long()
    x = cache[pages] if scale is None else cache.view(torch.uint8)[pages].view(cache.dtype)
    x = x.permute(0, 2, 1, 3, 4).float()
    x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])
    return x if scale is None else x * scale[:, None, None]


def run_decode(s):
    case = s["case"]
    if own:
        return package().decode_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], k_scale=s["k_scale"],
                                      v_scale=s["v_scale"], return_lse=case["lse"], sync=False)
    b, h, hk, d = s["q"].shape[0], case["heads"], case["kv_heads"], case["dim"]
    k = gathered(s["k_cache"], s["table"], s["k_scale"]).transpose(2, 3).contiguous()
    v = gathered(s["v_cache"], s["table"], s["v_scale"])
    scores = torch.matmul(s["q"].float().view(b, hk, h // hk, d) * d ** -0.5, k)
    visible = torch.arange(k.shape[3], device=DEVICE) < s["lens"][:, None, None, None]
    out, lse = softmax_times(scores, visible, v)
    out, lse = out.view(b, h, d).to(s["q"].dtype), lse.view(b, h)
    return (out, lse) if case["lse"] else out


def run_append(s):
    case = s["case"]
    if own:
        package().cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"],
                               k_scale=s["k_scale"], v_scale=s["v_scale"], sync=False)
        return s["k_cache"], s["v_cache"]
    token = torch.arange(s["k"].shape[0], dtype=torch.int32, device=DEVICE)
    of = torch.searchsorted(s["cu"][1:], token, right=True)
    position = (s["lens"][of] - s["cu"][of + 1] + token).long()
    page, slot = s["table"][of, position // case["page"]].long(), position % case["page"]
    return put(s["k"], s["k_cache"], page, slot, s["k_scale"]), put(s["v"], s["v_cache"], page, slot, s["v_scale"])


def put(x, cache, page, slot, scale):
    if scale is None:
        cache[page, :, slot] = x
    else:
        x = (x.float() / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
        cache.view(torch.uint8)[page, :, slot] = x.view(torch.uint8)
    return cache


# ---- what a pass cannot do without ------------------------------------------------------------------------
def work(case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        pairs = [(a, b) for a, b in zip(numbers(case["q_lens"]), k_lens_of(case))]
        seen = sum(a * b - a * (a - 1) // 2 for a, b in pairs)  # every listed and drawn prompt has as many keys as queries, or more
        return {"bytes": 2 * d * sum(2 * h * a + 2 * hk * b for a, b in pairs), "flops": 4 * d * h * seen}
    size = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "decode":
        lens = numbers(case["lens"])
        table = 4 * sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * hk * d * size * sum(lens) + 4 * h * d * len(lens) + table, "flops": 4 * d * h * sum(lens)}
    tokens = sum(numbers(case["new"]))
    return {"bytes": 2 * hk * d * (2 + size) * tokens, "flops": 0}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------
def attend(q, k, v, visible):
    """q [n, d], k and v [m, d], visible [n, m], all in 64 bits: (weighted values [n, d], log of the weights' sum [n])"""
    scores = torch.mm(q, k.t().contiguous()).div_(math.sqrt(q.shape[1]))
    scores[~visible] = -math.inf
    lse = torch.logsumexp(scores, 1)
    scores = torch.exp(scores - lse[:, None])
    scores[~visible] = 0.0
    return torch.mm(scores, v), lse


def exact(case, seed):
    s = prepare(case, seed)
    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "prompt":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        at_q, at_k = 0, 0
        for a, b in zip(numbers(case["q_lens"]), k_lens_of(case)):
            row = torch.arange(a, device=DEVICE)[:, None] + (b - a)
            visible = torch.arange(b, device=DEVICE)[None] <= row
            for n in range(h if a else 0):
                k, v = (s[x][at_k:at_k + b, n * hk // h].double() for x in ("k", "v"))
                out[at_q:at_q + a, n] = attend(s["q"][at_q:at_q + a, n].double(), k, v, visible)[0]
            at_q, at_k = at_q + a, at_k + b
        return out
    if case["op"] == "decode":
        lens = numbers(case["lens"])
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(lens):
            pages = s["table"][b, : -(-n // case["page"])].long()
            for g in range(hk if n else 0):
                k, v = (s[x][:, g].reshape(-1, case["page"], case["dim"]).view(torch.uint8)[pages].view(s[x].dtype)
                        .double().reshape(-1, case["dim"])[:n] for x in ("k_cache", "v_cache"))
                if s["k_scale"] is not None:
                    k, v = k * s["k_scale"][g].double(), v * s["v_scale"][g].double()
                mine = slice(g * h // hk, (g + 1) * h // hk)
                seen = torch.ones((h // hk, n), dtype=torch.bool, device=DEVICE)
                out[b, mine], lse[b, mine] = attend(s["q"][b, mine].double(), k, v, seen)
        return (out, lse) if case["lse"] else out
    got = []
    for new, old, scale in (("k", "k_cache", "k_scale"), ("v", "v_cache", "v_scale")):
        cache, x = s[old].double().contiguous(), s[new].double()
        if s[scale] is not None:
            x = nearest_e4m3(x / s[scale].double()[:, None])
        at = 0
        for b, (n, m) in enumerate(zip(numbers(case["new"]), numbers(case["before"]))):
            position = torch.arange(m, m + n, device=DEVICE)
            pages = s["table"][b][position // case["page"]].long()
            cache[pages, :, position % case["page"]] = x[at:at + n]
            at += n
        got.append(cache)
    return tuple(got)


def nearest_e4m3(x):
    """Nearest value of 4 exponent and 3 mantissa bits, ties to the even one, beyond the largest the largest."""
    x = x.clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step
