"""The paged key-value cache and the attention over it, as cases that can be timed and compared.

A host that serves several sequences at once keeps keys and values in pages of `ps` positions,
k and v [layers, n_pages, n_kv_heads, ps, head_dim], and one row of page numbers per sequence.
Kinds of case, one per operator:

  append   new K/V rows of packed sequences into their pages (tl_hip_launch_kv_append)
  copy     whole pages to other pages, K and V of every layer (tl_hip_launch_kv_copy_pages): the
           tail pages of forked sequences, and compaction
  decode   attention of one new token per sequence (tl_hip_launch_paged_attention_decode)
  prefill  causal attention of packed prompts, each over its own past
           (tl_hip_launch_paged_attention_prefill)

Where `own` is false everything is computed in its plain form with elementary torch operations.
Types are those of the library: f32 or f16 caches; f32 queries give f32 rows, f16 queries (over
f16 caches) f16 rows.  Sizes are those of the benchmark and the tests (4096-wide Llama layers: 32
heads over 8 KV heads of 128; TinyLlama: 32 over 4 of 64) and odd ones between.
"""
import ctypes
import math
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16}
CODE = {"f32": 0, "f16": 1}
SIZE = {"f32": 4, "f16": 2}
EXTRA = 3  # rows behind the last sequence of a padded batch


def listed():
    return [
        # one new token of 16 chats, rows as the linear layers write them (f32) into f16 pages
        {"name": "append_step", "kind": "append", "batch": 16, "tokens": 16, "past": 2000, "hkv": 8, "d": 128, "ps": 64, "new": "f32", "kv": "f16"},
        # packed prompts of 8192 tokens
        {"name": "append_prompts", "kind": "append", "batch": 8, "tokens": 8192, "past": 0, "hkv": 8, "d": 128, "ps": 64, "new": "f32", "kv": "f16"},
        # eight forked chats of a 22-layer TinyLlama get tail pages of their own
        {"name": "copy_fork", "kind": "copy", "pairs": 8, "layers": 22, "hkv": 4, "d": 64, "ps": 64, "kv": "f16"},
        # compaction of a pool after half of its sequences ended
        {"name": "copy_compact", "kind": "copy", "pairs": 768, "layers": 1, "hkv": 8, "d": 128, "ps": 64, "kv": "f16"},
        # a single chat at 512 cached positions: the smallest attention call
        {"name": "decode_one", "kind": "decode", "batch": 1, "len": 512, "ragged": False, "hq": 32, "hkv": 8, "d": 128, "ps": 64, "q": "f32", "kv": "f16"},
        # a serving batch of ragged lengths
        {"name": "decode_batch", "kind": "decode", "batch": 32, "len": 8192, "ragged": True, "hq": 32, "hkv": 8, "d": 128, "ps": 64, "q": "f32", "kv": "f16"},
        # two very long contexts: few rows, much cache
        {"name": "decode_long", "kind": "decode", "batch": 2, "len": 131072, "ragged": True, "hq": 32, "hkv": 8, "d": 128, "ps": 256, "q": "f16", "kv": "f16"},
        # TinyLlama chats over an f32 cache, small pages
        {"name": "decode_f32", "kind": "decode", "batch": 8, "len": 2048, "ragged": True, "hq": 32, "hkv": 4, "d": 64, "ps": 16, "q": "f32", "kv": "f32"},
        # chat turns of a few tokens each over their pasts
        {"name": "prefill_turns", "kind": "prefill", "batch": 6, "tokens": 75, "past": 2000, "hq": 32, "hkv": 4, "d": 64, "ps": 64, "q": "f32", "kv": "f16"},
        # packed prompts, rows as the linear layers write them (f32)
        {"name": "prefill_prompts", "kind": "prefill", "batch": 7, "tokens": 4001, "past": 0, "hq": 32, "hkv": 8, "d": 128, "ps": 64, "q": "f32", "kv": "f16"},
        # a long prompt in its second chunk, f16 throughout
        {"name": "prefill_long", "kind": "prefill", "batch": 1, "tokens": 8192, "past": 8192, "hq": 32, "hkv": 8, "d": 128, "ps": 128, "q": "f16", "kv": "f16"},
        # prompts over an f32 cache
        {"name": "prefill_f32", "kind": "prefill", "batch": 3, "tokens": 1100, "past": 0, "hq": 32, "hkv": 4, "d": 64, "ps": 32, "q": "f32", "kv": "f32"},
    ]


def draw(rng):
    """One more case of the same ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "copy", "decode", "decode", "prefill", "prefill"])
    c = {"kind": kind, "hkv": rng.choice([1, 2, 4, 8]), "d": rng.choice([64, 80, 96, 128, 128, 256]),
         "ps": rng.choice([16, 32, 64, 128, 256]), "kv": rng.choice(["f16", "f16", "f32"])}
    if kind == "append":
        batch = log(1, 64)
        c.update(batch=batch, tokens=batch + rng.choice([0, log(1, 8000)]), past=rng.choice([0, log(1, 4000)]), new=rng.choice(["f32", "f32", c["kv"]]))
        return c
    if kind == "copy":
        page = 2 * c["hkv"] * c["ps"] * c["d"] * SIZE[c["kv"]]
        layers = rng.choice([1, 1, 22])
        c.update(layers=layers, pairs=max(1, min(log(1, 768), (200 << 20) // (page * layers))))
        return c
    g = rng.choice([1, 3, 4, 4, 7, 8, 8, 16])
    c.update(hq=c["hkv"] * g, q=rng.choice(["f32", "f16"]) if c["kv"] == "f16" else "f32")
    row = c["hkv"] * c["d"] * SIZE[c["kv"]]
    if kind == "decode":
        batch = log(1, 64)
        most = min(131072, (300 << 20) // (row * batch))  # K or V of all sequences
        c.update(batch=batch, len=log(1, most), ragged=rng.random() < 0.7)
        return c
    tokens = log(1, 8192 if c["q"] == "f16" else 4096 if c["kv"] == "f16" else 1200)
    most = int(1.5e11 / (4 * c["hq"] * c["d"]) / (1 if c["kv"] == "f16" else 8))  # (query, key) pairs
    past = rng.choice([0, 0, log(1, 8192)])
    while tokens > 1 and tokens * (past + tokens) > most:
        tokens, past = -(-tokens // 2), past // 2
    c.update(batch=min(tokens, log(1, 8)), tokens=tokens, past=past)
    return c


# ------------------------------------------------------------------------ lengths ----
def lengths(case):
    """New tokens and total length of each sequence: the case's own numbers, whatever the seed."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    b = case["batch"]
    if case["kind"] == "decode":
        kv = [r.randint(1, case["len"]) if case["ragged"] else case["len"] for _ in range(b)]
        kv[r.randrange(b)] = case["len"]
        return [1] * b, kv
    cuts = sorted(r.sample(range(1, case["tokens"]), b - 1))
    new = [y - x for x, y in zip([0] + cuts, cuts + [case["tokens"]])]
    past = [r.randint(0, case["past"]) for _ in range(b)]
    past[r.randrange(b)] = case["past"]
    return new, [n + p for n, p in zip(new, past)]


def pairs_of(case):
    """(query, key) pairs that the causal mask leaves."""
    new, kv = lengths(case)
    return sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, kv))


# ------------------------------------------------------------------------- inputs ----
def generator(case, seed):
    g = torch.Generator(device="cuda")
    key = random.Random(repr((int(seed), sorted((k, v) for k, v in case.items() if k != "name")))).getrandbits(60)
    g.manual_seed(key)
    return g


def normal(g, dtype, *shape):
    return torch.empty(*shape, device="cuda", dtype=DTYPE[dtype]).normal_(generator=g)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, kind, ps, d = generator(case, seed), case["kind"], case["ps"], case["d"]
    s = {"case": case}
    if kind == "copy":
        n = 2 * case["pairs"]
        s["k"], s["v"] = (normal(g, case["kv"], case["layers"], n, case["hkv"], ps, d) for _ in range(2))
        order = torch.randperm(n, generator=g, device="cuda").tolist()
        s["src"], s["dst"] = (ctypes.c_int32 * (n // 2))(*order[: n // 2]), (ctypes.c_int32 * (n // 2))(*order[n // 2:])
        return s
    new, kv = lengths(case)
    need = [-(-t // ps) for t in kv]
    stride = max(need)
    n_pages = sum(need) + 2
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    # row b of the table: its pages, then whatever stood there before
    first = [0]
    for n in need:
        first.append(first[-1] + n)
    at = (ints(first[:-1])[:, None] + ints(list(range(stride)))[None]).clamp_(max=n_pages - 1)
    s["table"] = order[at.long()].contiguous()
    s["k"], s["v"] = (normal(g, case["kv"], n_pages, case["hkv"], ps, d) for _ in range(2))
    s["kv_lens"] = ints(kv)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["cu"] = ints(starts)
    s.update(n_pages=n_pages, stride=stride, most_new=max(new), most_kv=max(kv))
    rows = starts[-1] + (EXTRA if kind != "decode" else 0)
    s["rows"] = rows
    if kind == "append":
        # the K and V columns of a fused [k | v] projection: rows further apart than they are long
        s["kv_new"] = normal(g, case["new"], rows, 2, case["hkv"], d)
    else:
        s["q"] = normal(g, case["q"], rows, case["hq"], d)
        s["out"] = torch.full_like(s["q"], 0.5)
        s["scale"] = 1 / math.sqrt(d)
    return s


# --------------------------------------------------------------------- plain forms ----
def sequence_of(s):
    """For every row of the packed batch: its sequence and its index there; rows behind the last
    sequence have index -1."""
    t = torch.arange(s["rows"], device="cuda")
    cu = s["cu"].long()
    b = (t[:, None] >= cu[None, 1:]).sum(1)
    inside = t < cu[-1]
    b = b.clamp(max=cu.numel() - 2)
    return b, torch.where(inside, t - cu[b], -1)


def plain_append(s):
    c = s["case"]
    cu, lens = s["cu"].long(), s["kv_lens"].long()
    n = s["rows"] - EXTRA
    b, i = sequence_of(s)
    b, i = b[:n], i[:n]
    pos = lens[b] - (cu[b + 1] - cu[b]) + i
    page, slot = s["table"].long()[b, pos // c["ps"]], pos % c["ps"]
    rows = s["kv_new"][:n].to(DTYPE[c["kv"]])
    s["k"][page, :, slot] = rows[:, 0]
    s["v"][page, :, slot] = rows[:, 1]
    return {"k": s["k"], "v": s["v"]}


def plain_copy(s):
    src, dst = (torch.tensor(list(s[i]), device="cuda") for i in ("src", "dst"))
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"k": s["k"], "v": s["v"]}


def gathered(s, pages):
    """[batch, n_kv_heads, positions, head_dim] in 32 bits, zeros past each length."""
    c = s["case"]
    x = pages[s["table"].long()].permute(0, 2, 1, 3, 4).flatten(2, 3).float()
    seen = torch.arange(x.shape[2], device="cuda")[None] < s["kv_lens"][:, None]
    return torch.where(seen[:, None, :, None], x, torch.zeros((), device="cuda"))


def plain_attention(s):
    c = s["case"]
    hkv, d = c["hkv"], c["d"]
    g, b = c["hq"] // hkv, c["batch"]
    cu, lens = s["cu"].long(), s["kv_lens"].long()
    new, most = cu[1:] - cu[:-1], s["most_new"]
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i[None]).clamp(max=s["rows"] - 1)
    q = s["q"][at].float().view(b, most, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, most * g, d)
    k, v = gathered(s, s["k"]), gathered(s, s["v"])
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    seen = torch.arange(k.shape[2], device="cuda")[None, None] <= (lens - new)[:, None, None] + i[None, :, None]
    seen = seen & (torch.arange(k.shape[2], device="cuda") < lens[:, None])[:, None]
    x = x.view(b, hkv, most, g, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x.view(b, hkv, most * g, -1), v).view(b, hkv, most, g, d) / x.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(b, most, c["hq"], d).to(s["q"].dtype)
    out = s["out"]
    inside = i[None] < new[:, None]
    out[at[inside]] = o[inside]
    return out


PLAIN = {"append": plain_append, "copy": plain_copy, "decode": plain_attention, "prefill": plain_attention}


# ------------------------------------------------------------------- the framework ----
_device = None


def device():
    global _device
    if _device is None:
        from tl_amd import HipDevice
        _device = HipDevice(0)
    return _device


def checked(rc):
    if rc:
        raise RuntimeError(device().lib.tl_hip_last_error().decode())


def own_append(s):
    c, x = s["case"], s["kv_new"]
    width = c["hkv"] * c["d"]
    checked(device().lib.tl_hip_launch_kv_append(
        x.data_ptr(), x.data_ptr() + width * SIZE[c["new"]], CODE[c["new"]], 2 * width, 2 * width,
        s["k"].data_ptr(), s["v"].data_ptr(), CODE[c["kv"]], s["n_pages"], c["ps"], c["hkv"], c["d"],
        s["table"].data_ptr(), s["stride"], s["cu"].data_ptr(), s["kv_lens"].data_ptr(), c["batch"], s["rows"], None))
    return {"k": s["k"], "v": s["v"]}


def own_copy(s):
    c = s["case"]
    page_bytes = c["hkv"] * c["ps"] * c["d"] * SIZE[c["kv"]]
    checked(device().lib.tl_hip_launch_kv_copy_pages(
        s["k"].data_ptr(), s["v"].data_ptr(), c["layers"], 2 * c["pairs"], page_bytes, s["src"], s["dst"], c["pairs"], None))
    return {"k": s["k"], "v": s["v"]}


def own_decode(s):
    c = s["case"]
    checked(device().lib.tl_hip_launch_paged_attention_decode(
        s["q"].data_ptr(), CODE[c["q"]], c["hq"] * c["d"], s["k"].data_ptr(), s["v"].data_ptr(), CODE[c["kv"]], s["n_pages"],
        c["ps"], c["hq"], c["hkv"], c["d"], s["table"].data_ptr(), s["stride"], s["kv_lens"].data_ptr(), c["batch"],
        s["out"].data_ptr(), s["scale"], None, 0, None))
    return s["out"]


def own_prefill(s):
    c = s["case"]
    checked(device().lib.tl_hip_launch_paged_attention_prefill(
        s["q"].data_ptr(), CODE[c["q"]], c["hq"] * c["d"], s["k"].data_ptr(), s["v"].data_ptr(), CODE[c["kv"]], s["n_pages"],
        c["ps"], c["hq"], c["hkv"], c["d"], s["table"].data_ptr(), s["stride"], s["cu"].data_ptr(), s["kv_lens"].data_ptr(),
        c["batch"], s["rows"], s["out"].data_ptr(), s["scale"], None, 0, None))
    return s["out"]


OWN = {"append": own_append, "copy": own_copy, "decode": own_decode, "prefill": own_prefill}


def run(s):
    return (OWN if own else PLAIN)[s["case"]["kind"]](s)


# ---------------------------------------------------------------------- the bounds ----
def work(case):
    kind, d = case["kind"], case["d"]
    if kind == "copy":
        return {"bytes": 4 * case["pairs"] * case["layers"] * case["hkv"] * case["ps"] * d * SIZE[case["kv"]], "flops": 0}
    new, kv = lengths(case)
    index = 4 * (2 * case["batch"] + 1 + sum(-(-t // case["ps"]) for t in kv))
    if kind == "append":
        return {"bytes": 2 * sum(new) * case["hkv"] * d * (SIZE[case["new"]] + SIZE[case["kv"]]) + index, "flops": 0}
    rows = 2 * sum(new) * case["hq"] * d * SIZE[case["q"]]
    return {"bytes": 2 * sum(kv) * case["hkv"] * d * SIZE[case["kv"]] + rows + index, "flops": 4 * case["hq"] * d * pairs_of(case)}


# -------------------------------------------------------------- the same in 64 bits ----
def exact(case, seed):
    """Attention from its definition, one sequence and KV head at a time; rows behind the last
    sequence keep what the buffer held.  What moves values only is compared exactly elsewhere."""
    if case["kind"] == "copy":
        return None
    s = prepare(case, seed)
    new, kv = lengths(case)
    table = s["table"].cpu()
    if case["kind"] == "append":
        return None if case["new"] == case["kv"] else exact_append(case, s, new, kv, table)
    d, g = case["d"], case["hq"] // case["hkv"]
    out, t = torch.full(s["q"].shape, 0.5, dtype=torch.float64, device="cuda"), 0
    for b, (n, total) in enumerate(zip(new, kv)):
        pages = table[b, : -(-total // case["ps"])].long().cuda()
        first = torch.arange(total - n, total, device="cuda")
        for h in range(case["hkv"]):
            k, v = (s[x][pages, h].reshape(-1, d)[:total].double() for x in ("k", "v"))
            for i in range(0, n, 1024):  # queries i .. i + 1023 with all heads of the group
                q = s["q"][t + i : t + min(n, i + 1024), h * g : (h + 1) * g].double()
                x = q.flatten(0, 1) @ k.T.contiguous() / math.sqrt(d)
                late = torch.arange(total, device="cuda")[None] > first[i : i + 1024].repeat_interleave(g)[:, None]
                x = torch.softmax(x.masked_fill_(late, -math.inf), -1)
                out[t + i : t + i + q.shape[0], h * g : (h + 1) * g] = (x @ v).view(q.shape)
        t += n
    return out


def exact_append(case, s, new, kv, table):
    k, v, t = s["k"].double(), s["v"].double(), 0
    for b, (n, total) in enumerate(zip(new, kv)):
        for j in range(total - n, total):
            page, slot = int(table[b, j // case["ps"]]), j % case["ps"]
            k[page, :, slot], v[page, :, slot] = s["kv_new"][t, 0].double(), s["kv_new"][t, 1].double()
            t += 1
    return {"k": k, "v": v}
