"""The operators that serve several sequences at once, as a user of this framework calls them, for measuring.

Three kinds of work, in the shapes of the repository's configurations (SmolLM2-135M, the
attention of Qwen2.5-0.5B, Qwen3-0.6B, TinyLlama-1.1B and Llama-3-8B):
  prompts   causal attention over packed prompts of different lengths, alone or behind a
            prefix that all of them share (one layer)
  answers   one new token of every sequence over the shared prefix and the sequence's own
            positions (one layer)
  logits    penalties for repeated tokens, biases and grammar masks on a batch's logits

q and the results are f32; the caches hold keys and values in f32 or bf16.  With `own` the
calls go to the framework's handles; without, the same results come from elementary torch
operations in 32 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"

# attention of the configurations: query heads, kv heads, head_dim
SHAPES = {
    "smollm2": (9, 3, 64),
    "qwen2.5": (14, 2, 64),
    "qwen3": (16, 8, 128),
    "tinyllama": (32, 4, 64),
    "llama3": (32, 8, 128),
}


def listed():
    return [
        # a few very short prompts of the smallest model: latency
        dict(name="prompts-smollm2-short", kind="prompts", shape="smollm2", type="f32", n=3, lo=1, hi=23, mix=1,
             prefix=0),
        # ordinary requests that arrive together, odd lengths
        dict(name="prompts-qwen2.5-8", kind="prompts", shape="qwen2.5", type="f32", n=8, lo=33, hi=701, mix=2,
             prefix=0),
        # long prompts of a large model: the largest prompt work
        dict(name="prompts-llama3-6", kind="prompts", shape="llama3", type="f32", n=6, lo=500, hi=2047, mix=3,
             prefix=0),
        # the same kind of batch on a 16-bit cache
        dict(name="prompts-llama3-6-bf16", kind="prompts", shape="llama3", type="bf16", n=6, lo=500, hi=2047, mix=4,
             prefix=0),
        # users' questions behind one system prompt
        dict(name="questions-qwen3-16", kind="prompts", shape="qwen3", type="f32", n=16, lo=12, hi=161, mix=5,
             prefix=1500),
        # four drafts of one short answer by the smallest model: latency
        dict(name="answers-smollm2-4", kind="answers", shape="smollm2", type="f32", n=4, lo=1, hi=60, mix=6,
             prefix=300),
        # sixteen users behind a system prompt with examples
        dict(name="answers-qwen2.5-16", kind="answers", shape="qwen2.5", type="f32", n=16, lo=20, hi=400, mix=7,
             prefix=4001),
        # a large model's samples over one long document
        dict(name="answers-llama3-32", kind="answers", shape="llama3", type="f32", n=32, lo=10, hi=900, mix=8,
             prefix=16384),
        # many samples over the longest document, 16-bit cache: the largest cache read
        dict(name="answers-llama3-64-bf16", kind="answers", shape="llama3", type="bf16", n=64, lo=100, hi=1500, mix=9,
             prefix=32768),
        # one answer's logits under penalties: latency
        dict(name="logits-49k-1", kind="logits", rows=1, vocab=49152, tokens=200, biases=8, masked=False, mix=10),
        # a small batch with long histories, biases and grammars over a large vocabulary
        dict(name="logits-152k-8", kind="logits", rows=8, vocab=151936, tokens=4000, biases=300, masked=True, mix=11),
        # a full batch of a large model under grammars
        dict(name="logits-128k-64", kind="logits", rows=64, vocab=128256, tokens=1500, biases=32, masked=True,
             mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompts", "prompts", "answers", "answers", "logits"])
    mix = rng.randrange(1 << 20)
    if kind == "logits":
        rows = _log(rng, 1, 64)
        vocab = rng.choice([32000, 49152, 128256, 151936, rng.randint(5001, 151935)])
        while rows * vocab > 64 * 128256:
            rows -= 1
        return dict(kind=kind, rows=rows, vocab=vocab, tokens=_log(rng, 1, 4000), biases=rng.choice([0, _log(rng, 1, 300)]),
                    masked=rng.random() < 0.6, mix=mix)
    shape, kv_type = rng.choice(sorted(SHAPES)), rng.choice(["f32", "f32", "bf16"])
    heads, kvh, d = SHAPES[shape]
    if kind == "prompts":
        n, hi = _log(rng, 1, 24), _log(rng, 4, 2048)
        prefix = 0 if rng.random() < 0.6 else _log(rng, 64, 4000)
        case = dict(kind=kind, shape=shape, type=kv_type, n=n, lo=max(1, hi // rng.choice([2, 8, 40])), hi=hi, mix=mix,
                    prefix=prefix)
        # within the largest listed prompts' work, padded to the longest or not
        while case["n"] > 1 and (case["n"] * hi * (hi + prefix) * heads * d > 6 * 2047 * 2047 * 32 * 128
                                 or work(case)["flops"] > 7.6e10 or work(case)["bytes"] > 2.8e8):
            case["n"] -= 1
        return case
    n, hi = _log(rng, 1, 64), _log(rng, 1, 1500)
    prefix = _log(rng, 100, 32768)
    # within the largest listed answers' work
    while prefix > 100 and n * heads * d * (prefix + hi) > 64 * 32 * 128 * 33000 or prefix * kvh * d > 16384 * 8 * 128 * (
            2 if kv_type == "bf16" else 1):
        prefix = prefix * 3 // 4
    return dict(kind=kind, shape=shape, type=kv_type, n=n, lo=max(1, hi // rng.choice([2, 10, 50])), hi=hi, mix=mix,
                prefix=prefix)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(case):
    """Each sequence's positions, its new tokens included: one of them the longest, the others
    spread over the range."""
    rng = random.Random(case["mix"])
    return [case["hi"]] + [_log(rng, case["lo"], case["hi"]) for _ in range(case["n"] - 1)]


def _starts_counts(case):
    """(first new position, new tokens) of every sequence: whole prompts, or the last position."""
    lens = _lengths(case)
    if case["kind"] == "prompts":
        return [0] * len(lens), lens
    return [x - 1 for x in lens], [1] * len(lens)


def _attention_inputs(case, seed):
    """The prefix's and the sequences' keys and values and the new tokens' queries.  Heads
    differ in how sharply they look (score deviations of 0.5 to 3)."""
    heads, kvh, d = SHAPES[case["shape"]]
    g = _gen(seed)
    lens = _lengths(case)
    starts, counts = _starts_counts(case)
    kv_type = torch.float32 if case["type"] == "f32" else torch.bfloat16
    total = sum(counts)
    q = torch.randn(total, heads, d, generator=g, device=DEV)
    q *= torch.exp(torch.rand(heads, 1, generator=g, device=DEV) * math.log(6.0)) * 0.5

    def cache(*shape):
        return torch.randn(*shape, d, generator=g, device=DEV).to(kv_type)

    return {"case": dict(case), "heads": heads, "kvh": kvh, "d": d, "lens": lens, "starts": starts, "counts": counts, "q": q,
            # [kv_head][position][d] of the prefix, [sequence][kv_head][position][d] of the others
            "pk": cache(kvh, case["prefix"]), "pv": cache(kvh, case["prefix"]),
            "k": cache(case["n"], kvh, max(lens)), "v": cache(case["n"], kvh, max(lens))}


def _logits_inputs(case, seed):
    """Logits as a language model's are (a broad normal body, a few likely ids), each row's tokens
    so far (some of them often), its settings, its biases and its grammar's allowed ids as bits."""
    rows, vocab = case["rows"], case["vocab"]
    g = _gen(seed)
    rng = random.Random(case["mix"])
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.5
    hot = torch.randint(0, vocab, (rows, 12), generator=g, device=DEV)
    x.scatter_add_(1, hot, torch.rand(rows, 12, generator=g, device=DEV) * 4 + 4)
    tokens = (torch.rand(rows, case["tokens"], generator=g, device=DEV) ** 4 * vocab).to(torch.int32)
    n_tokens = [case["tokens"]] + [rng.randint(0, case["tokens"]) for _ in range(rows - 1)]
    n_prompt = [rng.randint(0, n) for n in n_tokens]
    n_bias = [rng.randint(0, case["biases"]) for _ in range(rows)] if case["biases"] else [0] * rows
    start = torch.tensor([sum(n_bias[:r]) for r in range(rows + 1)], dtype=torch.int32, device=DEV)
    # each row's ids differ from one another: one of every stretch of the vocabulary
    span = vocab // max(1, case["biases"])
    place = torch.cat([torch.arange(n, device=DEV) for n in n_bias]) if sum(n_bias) else torch.zeros(0, device=DEV)
    bias_ids = (place * span + (torch.rand(sum(n_bias), generator=g, device=DEV) * span).long()).to(torch.int32)
    state = {"case": dict(case), "x": x, "tokens": tokens, "out": torch.empty_like(x),
             "n_tokens": torch.tensor(n_tokens, dtype=torch.int32, device=DEV),
             "n_prompt": torch.tensor(n_prompt, dtype=torch.int32, device=DEV),
             "repetition": torch.rand(rows, generator=g, device=DEV) * 0.4 + 1,
             "presence": torch.rand(rows, generator=g, device=DEV) * 1.5,
             "frequency": torch.rand(rows, generator=g, device=DEV) * 0.5,
             "bias_start": start, "bias_ids": bias_ids,
             "bias": torch.randn(sum(n_bias), generator=g, device=DEV) * 4, "mask": None}
    if case["masked"]:
        # some grammars allow much of the vocabulary, some a few ids
        words = (vocab + 31) // 32
        share = torch.rand(rows, 1, generator=g, device=DEV) ** 2
        bits = torch.rand(rows, words * 32, generator=g, device=DEV) < share
        weight = 2 ** torch.arange(32, device=DEV, dtype=torch.int64)
        w = (bits.view(rows, words, 32).long() * weight).sum(-1)
        state["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    return state


_stream = None


def _program_stream():
    """The program's stream: what it queues runs in order, one call after another."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream


def _batch(s):
    """The batch that a serving program keeps: the caches filled, the step planned."""
    from wick_amd.batch import DeviceBatch
    case, kvd = s["case"], s["kvh"] * s["d"]
    b = DeviceBatch(layers=1, heads=s["heads"], kv_heads=s["kvh"], head_dim=s["d"], sequences=case["n"],
                    capacity=max(s["lens"]), prefix_capacity=case["prefix"], max_tokens=sum(s["lens"]), dtype=case["type"])
    b.set_stream(_program_stream().cuda_stream)

    def rows(c, n):  # [kv_head][position][d] -> [position][kv_head * d]
        return c[:, :n].permute(1, 0, 2).reshape(n, kvd).float()

    if case["prefix"]:
        k, v = (rows(s[name], case["prefix"]).contiguous() for name in ("pk", "pv"))
        torch.cuda.synchronize()
        b.write_prefix_device(0, 0, case["prefix"], k.data_ptr(), v.data_ptr())
        b.synchronize()
    k, v = (torch.cat([rows(c, n) for c, n in zip(s[name], s["lens"])]).contiguous() for name in ("k", "v"))
    torch.cuda.synchronize()
    b.plan([0] * case["n"], s["lens"], case["prefix"])
    b.append_device(0, k.data_ptr(), v.data_ptr())
    b.plan(s["starts"], s["counts"], case["prefix"])
    b.synchronize()
    return b


def prepare(case, seed):
    if case["kind"] == "logits":
        s = _logits_inputs(case, seed)
        if own:  # the program's stream does not wait for the one that makes the inputs
            torch.cuda.synchronize()
        return s
    s = _attention_inputs(case, seed)
    s["att"] = torch.empty_like(s["q"])
    if own:
        s["batch"] = _batch(s)
    # the rows of the packed tokens in a batch padded to the longest, and back
    widest = max(s["counts"])
    s["row"] = torch.cat([torch.arange(t, device=DEV) + i * widest for i, t in enumerate(s["counts"])])
    s["start"] = torch.tensor(s["starts"], device=DEV)
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    if s["case"]["kind"] == "logits":
        return _run_logits(s)
    if own:
        s["batch"].attention_device(0, s["q"].data_ptr(), s["att"].data_ptr())
        return s["att"]
    n, kvh, heads, d = s["case"]["n"], s["kvh"], s["heads"], s["d"]
    group, widest, prefix = heads // kvh, max(s["counts"]), s["case"]["prefix"]
    q = s["q"].new_zeros(n * widest, heads, d)
    q[s["row"]] = s["q"] / math.sqrt(d)
    # the sequences' own positions, [sequence][kv_head][group * token][position]
    q = q.view(n, widest, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * widest, d)
    own_scores = torch.matmul(q, s["k"].float().transpose(2, 3).contiguous())
    length = own_scores.shape[3]
    token = torch.arange(widest, device=DEV)
    seen = torch.arange(length, device=DEV) <= (s["start"][:, None] + token)[:, :, None]
    own_scores = own_scores.view(n, kvh, group, widest, length).masked_fill_(~seen[:, None, None], -math.inf)
    own_scores = own_scores.view(n, kvh, group * widest, length)
    top = own_scores.amax(-1, keepdim=True)
    if prefix:
        # the prefix, all sequences' rows at once, [kv_head][sequence * group * token][position]
        qp = q.transpose(0, 1).reshape(kvh, n * group * widest, d)
        prefix_scores = torch.matmul(qp, s["pk"].float().transpose(1, 2).contiguous())
        prefix_top = prefix_scores.amax(-1).view(kvh, n, group * widest).transpose(0, 1)[..., None]
        top = torch.maximum(top, prefix_top)
    p = (own_scores - top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, s["v"].float())
    if prefix:
        flat = top.transpose(0, 1).reshape(kvh, n * group * widest, 1)
        p = (prefix_scores - flat).exp_()
        total = total + p.sum(-1).view(kvh, n, group * widest).transpose(0, 1)[..., None]
        out = out + torch.matmul(p, s["pv"].float()).view(kvh, n, group * widest, d).transpose(0, 1)
    out = (out / total).view(n, kvh, group, widest, d).permute(0, 3, 1, 2, 4)
    return out.reshape(n * widest, heads, d)[s["row"]]


def _run_logits(s):
    x, rows, vocab = s["x"], s["case"]["rows"], s["case"]["vocab"]
    if own:
        from wick_amd.logits import adjust_logits_device
        adjust_logits_device(s["x"].data_ptr(), rows, vocab, s["out"].data_ptr(), repetition=s["repetition"].data_ptr(),
                             presence=s["presence"].data_ptr(), frequency=s["frequency"].data_ptr(),
                             tokens=s["tokens"].data_ptr(), tokens_stride=s["tokens"].shape[1],
                             n_tokens=s["n_tokens"].data_ptr(), n_prompt=s["n_prompt"].data_ptr(),
                             bias_start=s["bias_start"].data_ptr(), bias_ids=s["bias_ids"].data_ptr(),
                             bias=s["bias"].data_ptr(), n_bias=s["bias"].numel(),
                             mask=None if s["mask"] is None else s["mask"].data_ptr(),
                             masks=rows, stream=_program_stream().cuda_stream)
        return s["out"]
    place = torch.arange(s["tokens"].shape[1], device=DEV)
    held = place < s["n_tokens"][:, None]
    written = held & (place >= s["n_prompt"][:, None])
    ids = s["tokens"].long()
    seen = torch.zeros_like(x).scatter_add_(1, ids, held.float())
    count = torch.zeros_like(x).scatter_add_(1, ids, written.float())
    r = s["repetition"][:, None]
    y = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    y = y - (s["frequency"][:, None] * count + torch.where(count > 0, s["presence"][:, None], 0.0))
    if s["bias"].numel():
        row = torch.repeat_interleave(torch.arange(rows, device=DEV), (s["bias_start"][1:] - s["bias_start"][:-1]).long(),
                                      output_size=s["bias"].numel())
        y[row, s["bias_ids"].long()] += s["bias"]
    if s["mask"] is not None:
        i = torch.arange(vocab, device=DEV)
        allowed = (s["mask"][:, i // 32] >> (i % 32)) & 1
        y = torch.where(allowed != 0, y, -math.inf)
    return y


# ---------------------------------------------------------------- the work, and the values


def work(case):
    if case["kind"] == "logits":
        words = (case["vocab"] + 31) // 32 if case["masked"] else 0
        per_row = 8 * case["vocab"] + 4 * words + 2 * case["tokens"] + 4 * case["biases"]
        return {"bytes": case["rows"] * per_row, "flops": 6 * case["rows"] * case["vocab"]}
    heads, kvh, d = SHAPES[case["shape"]]
    size = 4 if case["type"] == "f32" else 2
    starts, counts = _starts_counts(case)
    pairs = sum(t * (case["prefix"] + a) + t * (t + 1) // 2 for a, t in zip(starts, counts))
    positions = case["prefix"] + sum(a + t for a, t in zip(starts, counts))
    return {"bytes": 2 * size * kvh * d * positions + 8 * heads * d * sum(counts), "flops": 4 * d * heads * pairs}


def exact(case, seed):
    return _exact_logits(case, seed) if case["kind"] == "logits" else _exact_attention(case, seed)


def _exact_attention(case, seed):
    """softmax(q k / sqrt(d)) v of one sequence and kv head after the other, in 64 bits."""
    s = _attention_inputs(case, seed)
    group, d, prefix = s["heads"] // s["kvh"], s["d"], case["prefix"]
    out = torch.empty(sum(s["counts"]), s["heads"], d, dtype=torch.float64, device=DEV)
    at = 0
    for i, (a, t) in enumerate(zip(s["starts"], s["counts"])):
        position = torch.arange(prefix + a + t, device=DEV)
        hidden = position[None, :] > prefix + a + torch.arange(t, device=DEV)[:, None]
        for h in range(s["kvh"]):
            keys = torch.cat([s["pk"][h], s["k"][i, h, :a + t]]).double()
            values = torch.cat([s["pv"][h], s["v"][i, h, :a + t]]).double()
            for j in range(h * group, (h + 1) * group):
                w = s["q"][at:at + t, j].double() @ keys.t() / math.sqrt(d)
                w[hidden] = -math.inf
                out[at:at + t, j] = torch.softmax(w, -1) @ values
        at += t
    return out


def _exact_logits(case, seed):
    """Each row's rules applied to its logits in their order, in 64 bits."""
    s = _logits_inputs(case, seed)
    y = s["x"].double()
    for r in range(case["rows"]):
        n, first = int(s["n_tokens"][r]), int(s["n_prompt"][r])
        ids = s["tokens"][r, :n].long()
        seen = ids.unique()
        old = y[r, seen]
        by = s["repetition"][r].double()
        y[r, seen] = torch.where(old > 0, old / by, old * by)
        written, count = ids[first:].unique(return_counts=True)
        y[r, written] -= s["frequency"][r].double() * count + s["presence"][r].double()
        a, b = int(s["bias_start"][r]), int(s["bias_start"][r + 1])
        y[r, s["bias_ids"][a:b].long()] += s["bias"][a:b].double()
        if s["mask"] is not None:
            words = s["mask"][r].cpu().numpy().view("uint32")
            bits = torch.from_numpy(words.astype("int64"))[:, None] >> torch.arange(32) & 1
            y[r, bits.flatten()[:case["vocab"]].to(DEV) == 0] = -math.inf
    return y
