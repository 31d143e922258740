"""Measured cases of the attention side of a decoder layer: norms of queries and keys per head with the position
rotation, the 8-bit key/value cache as it is written and read back, and attention over that cache.

``own`` false: the plain forms, elementary torch operations in 32 bits.  ``own`` true: the calls of ollama_amd.qmm on the
same buffers.  The cache is one block of device memory in the layout that include/mi_qmm.h states for mi_qmm_kv_create;
both forms work on it directly, so nothing has to be converted for either.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64  # tokens of a cache page
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}  # ggml type ids
PER127 = float(np.float32(1.0 / 127.0))  # a block's scale is its largest magnitude times this, rounded to fp32


def listed():
    return [
        # one token of one conversation: 32 query and 8 key heads of 128, normed per head, far into a long context
        dict(name="rope_token", op="rope", rows=1, heads=32, kv_heads=8, dim=128, rot=128, pairs="halves", norm=True, type="f32",
             base=1e6, far=131072),
        # a mixed step of many heads of 64: some tokens of prompts and some single ones, adjacent pairs, fp16 activations
        dict(name="rope_mixed", op="rope", rows=333, heads=64, kv_heads=8, dim=64, rot=64, pairs="adjacent", norm=False, type="f16",
             base=150000.0, far=40000),
        # the prompts of a prefill step
        dict(name="rope_prompt", op="rope", rows=8192, heads=32, kv_heads=8, dim=128, rot=128, pairs="halves", norm=True, type="f32",
             base=5e5, far=8192),
        # a decode step of 64 conversations: one token each goes into the cache, in the middle of a block of tokens
        dict(name="kv_step", op="write", seqs=64, new=1, kv=4096, kv_heads=8, dim=128, block=64, type="f32"),
        # chunks of four prompts that go on in partly filled pages
        dict(name="kv_prompt", op="write", seqs=4, new=2048, kv=4500, kv_heads=8, dim=128, block=32, type="f32"),
        # three short conversations of a model with heads of 80, read back for a check or a transfer
        dict(name="kv_read_small", op="read", seqs=3, new=0, kv=777, kv_heads=5, dim=80, block=16, type="f16"),
        # one long context read back whole
        dict(name="kv_read_long", op="read", seqs=1, new=0, kv=65536, kv_heads=8, dim=128, block=64, type="bf16"),
        # the next token of one conversation
        dict(name="attend_token", op="attend", seqs=1, new=1, kv=4096, heads=32, kv_heads=8, dim=128, block=64, type="f32",
             window=0, cap=0.0, sinks=False),
        # a decode step of 64 conversations of different lengths
        dict(name="attend_batch", op="attend", seqs=64, new=1, kv=8192, heads=32, kv_heads=8, dim=128, block=32, type="f32",
             window=0, cap=0.0, sinks=False),
        # a decode step through a sliding window with a learned sink per head, 64 heads of 64
        dict(name="attend_window", op="attend", seqs=33, new=1, kv=4000, heads=64, kv_heads=8, dim=64, block=64, type="f16",
             window=128, cap=0.0, sinks=True),
        # the prefill of two prompts
        dict(name="attend_prompt", op="attend", seqs=2, new=4096, kv=4096, heads=32, kv_heads=8, dim=128, block=64, type="bf16",
             window=0, cap=0.0, sinks=False),
        # a chunk of a long prompt over what the cache holds of it, heads of 256 with capped scores
        dict(name="attend_chunk", op="attend", seqs=1, new=509, kv=16001, heads=16, kv_heads=8, dim=256, block=64, type="f32",
             window=0, cap=50.0, sinks=False),
    ]


def _between(rng, lo, hi):
    """a whole number of lo..hi, spread over its logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attend", "attend"])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 80, 96, 128, 256])
    kind = rng.choice(["f32", "f16", "bf16"])
    block = rng.choice([16, 32, 64])
    if op == "rope":
        rows = min(_between(rng, 1, 8192), 8192 * 5120 // ((group + 1) * kv_heads * dim))
        return dict(op=op, rows=rows, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim // 2]),
                    pairs=rng.choice(["halves", "adjacent"]), norm=rng.random() < 0.5, type=kind, base=rng.choice([1e4, 5e5, 1e6]),
                    far=_between(rng, rows, 131072))
    if op == "attend":
        if rng.random() < 0.6:  # a decode step: up to four tokens each
            new, kv = rng.randint(1, 4), _between(rng, 8, 8192)
            seqs = min(_between(rng, 1, 64), max(1, 64 * 8192 * 8 * 128 // (kv * kv_heads * dim)))
        else:  # prompts, or chunks of them
            new = _between(rng, 16, 2048)
            kv, seqs = _between(rng, new, 8192), rng.randint(1, 2)
            new = max(1, min(new, 180 * 10 ** 9 // (4 * seqs * kv * group * kv_heads * dim)))
        return dict(op=op, seqs=seqs, new=min(new, kv), kv=kv, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, block=block,
                    type=kind, window=rng.choice([0, 0, 100, 128, 1024]), cap=rng.choice([0.0, 0.0, 30.0]), sinks=rng.random() < 0.3)
    seqs = _between(rng, 1, 64)
    kv = _between(rng, 1, max(64, min(65536, 65536 * 8 * 128 // (seqs * kv_heads * dim))))
    if op == "read":
        return dict(op=op, seqs=seqs, new=0, kv=kv, kv_heads=kv_heads, dim=dim, block=block, type=kind)
    new = min(_between(rng, 1, kv), max(1, 8192 * 8 * 128 // (seqs * kv_heads * dim)))
    return dict(op=op, seqs=seqs, new=new, kv=kv, kv_heads=kv_heads, dim=dim, block=block, type=kind)


# ---- what a case consists of ------------------------------------------------------------------------------------------
def _lengths(case):
    """(new rows, tokens in the cache) of each sequence: ragged, the first ones the full lengths"""
    new, kv = [], []
    for i in range(case["seqs"]):
        f = 1.0 - 0.6 * ((i * 0.6180339887) % 1.0)
        kv.append(max(1, int(case["kv"] * f)))
        n = case["new"] if case["new"] <= 4 else max(1, int(case["new"] * f))
        new.append(min(n, kv[-1]) if case["op"] != "read" else kv[-1])
    return new, kv


def _row_dim(dim):
    return (dim + 63) // 64 * 64


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["op"] == "rope":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * size + 4 * case["rows"], "flops": (4 * case["norm"] + 3) * values}
    new, kv = _lengths(case)
    token = 2 * case["kv_heads"] * case["dim"]  # values of a token's key and value
    if case["op"] == "read":
        return {"bytes": sum(kv) * token * (1 + size) + 8 * case["kv_heads"] * sum(-(-t // case["block"]) for t in kv), "flops": sum(kv) * token}
    if case["op"] == "write":  # the new rows in, their codes out; then the blocks they touch read back
        b = case["block"]
        back = sum(t - (t - n) // b * b for n, t in zip(new, kv))
        old = back - sum(new)
        return {"bytes": sum(new) * token * (size + 1) + old * token + back * token * (1 + size), "flops": 3 * sum(new) * token + back * token}
    pairs = seen = 0
    for n, t in zip(new, kv):
        w = case["window"] or t
        pos = np.arange(t - n, t, dtype=np.int64)
        pairs += int(np.minimum(pos + 1, w).sum())
        seen += t - max(0, t - n + 1 - w)
    return {"bytes": seen * token + 2 * sum(new) * case["heads"] * case["dim"] * size, "flops": 4 * pairs * case["heads"] * case["dim"]}


_ctx = None


def _context():
    """the library's context, on the stream torch works on"""
    global _ctx
    from ollama_amd import qmm

    if _ctx is None:
        _ctx = qmm.Context(torch.cuda.current_device())
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream or qmm.STREAM_LEGACY)
    return _ctx


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kind, dim = TYPES[case["type"]], case["dim"]
    s = {"case": case}
    if case["op"] == "rope":
        n, h, kh = case["rows"], case["heads"], case["kv_heads"]
        s["q"] = (rnd(n, h, dim) * 2).to(kind)
        s["k"] = (rnd(n, kh, dim) * 2).to(kind)
        s["q_weight"] = 1 + 0.2 * rnd(dim) if case["norm"] else None
        s["k_weight"] = 1 + 0.2 * rnd(dim) if case["norm"] else None
        s["pos"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda", dtype=torch.int32)
        half = case["rot"] // 2
        s["freqs"] = torch.tensor([case["base"] ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        if own:  # the description of the heads, which a program keeps
            from ollama_amd import qmm

            s["heads"] = qmm.QKHeads(GGML[case["type"]], h, kh, dim, s["freqs"].data_ptr(), case["rot"],
                                     qmm.ROPE_HALVES if case["pairs"] == "halves" else qmm.ROPE_ADJACENT,
                                     q_weight=s["q_weight"].data_ptr() if case["norm"] else None,
                                     k_weight=s["k_weight"].data_ptr() if case["norm"] else None, eps=1e-6)
        return s
    new, kv = _lengths(case)
    seqs, kh, b, dp = len(kv), case["kv_heads"], case["block"], _row_dim(dim)
    table = -(-max(kv) // PAGE)
    pages = seqs * table + 3
    s["pages"] = torch.randperm(pages, generator=g, device="cuda")[: seqs * table].to(torch.int32).reshape(seqs, table).contiguous()
    starts = [0] + np.cumsum(new).tolist()
    s["row_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["new"], s["rows"], s["kv_rows"] = new, starts[-1], kv
    # the cache's memory: key codes, value codes (a byte holds the code plus 128), key scales, value scales
    codes, scales = pages * kh * PAGE * dp, pages * kh * (PAGE // b)
    mem = torch.empty(2 * codes + 8 * scales, dtype=torch.uint8, device="cuda")
    s["memory"] = mem
    for name, at in (("k_codes", 0), ("v_codes", codes)):
        c = mem[at:at + codes]
        for i in range(0, codes, 1 << 26):  # normal values, 127 the largest, plus 128; in pieces, since the normals are four times as large
            part = c[i:i + (1 << 26)]
            part.copy_((rnd(part.numel()) * 36).clamp_(-127, 127).round_().add_(128))
        s[name] = c
    for name, at in (("k_scale", 2 * codes), ("v_scale", 2 * codes + 4 * scales)):
        t = mem[at:at + 4 * scales].view(torch.float32)
        t.copy_((torch.rand(scales, generator=g, device="cuda") * 0.8 + 0.6) * (3.5 / 127))
        s[name] = t.view(pages, kh, PAGE // b)
    if case["op"] == "attend":
        s["q"] = (rnd(s["rows"], case["heads"], dim) * 1.5).to(kind)
        s["sinks"] = rnd(case["heads"]) if case["sinks"] else None
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = dim ** -0.5
    else:
        back = new if case["op"] == "read" else [t - (t - n) // b * b for n, t in zip(new, kv)]
        s["back"] = back
        ends = [0] + np.cumsum(back).tolist()
        s["back_start"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s["k_back"] = torch.empty(ends[-1], kh, dim, dtype=kind, device="cuda")
        s["v_back"] = torch.empty_like(s["k_back"])
        if case["op"] == "write":
            s["k"], s["v"] = rnd(s["rows"], kh, dim).to(kind), rnd(s["rows"], kh, dim).to(kind)
    if own:  # the handles that a program keeps: the cache over its memory, the step's sequences, the attention's description
        from ollama_amd import qmm

        s["kv"] = _context().kv_create(pages, kh, dim, b, memory=mem.data_ptr())
        s["batch"] = qmm.Batch(seqs, table, s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["pages"].data_ptr())
        if case["op"] == "attend":
            s["how"] = qmm.Attention(GGML[case["type"]], case["heads"], s["scale"], window=case["window"], softcap=case["cap"],
                                     sinks=s["sinks"].data_ptr() if case["sinks"] else None)
        else:
            s["back_batch"] = qmm.Batch(seqs, table, s["back_start"].data_ptr(), s["kv_len"].data_ptr(), s["pages"].data_ptr())
    return s


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[op](s)
    c, kind = _context(), GGML[s["case"]["type"]]
    if op == "rope":
        c.qk_norm_rope_device(s["heads"], s["q"].data_ptr(), s["k"].data_ptr(), s["pos"].data_ptr(), s["case"]["rows"],
                              s["q_out"].data_ptr(), s["k_out"].data_ptr())
        return s["q_out"], s["k_out"]
    if op == "attend":
        c.attention_device(s["kv"], s["batch"], s["how"], s["q"].data_ptr(), s["rows"], s["out"].data_ptr())
        return s["out"]
    if op == "write":
        c.kv_write_device(s["kv"], s["batch"], kind, s["k"].data_ptr(), s["v"].data_ptr(), s["rows"])
    c.kv_read_device(s["kv"], s["back_batch"], kind, s["k_back"].data_ptr(), s["v_back"].data_ptr(), s["k_back"].shape[0])
    return (s["k_back"], s["v_back"], s["k_scale"], s["v_scale"]) if op == "write" else (s["k_back"], s["v_back"])


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _plain_rope(s):
    case = s["case"]
    turn = s["pos"].to(torch.float64)[:, None] * s["freqs"][None, :]  # angles of far positions: 64 bits
    cos, sin = turn.cos().to(torch.float32)[:, None, :], turn.sin().to(torch.float32)[:, None, :]
    rot, half = case["rot"], case["rot"] // 2
    at = torch.arange(half, device="cuda")
    first, second = (at, at + half) if case["pairs"] == "halves" else (2 * at, 2 * at + 1)

    def one(x, weight):
        y = x.to(torch.float32)
        if weight is not None:
            y = y * (1.0 / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * weight
        z = y.clone()
        a, b = y[..., first], y[..., second]
        z[..., first] = a * cos - b * sin
        z[..., second] = a * sin + b * cos
        return z.to(x.dtype)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def _key_values(codes, kh, dp):
    """key codes of pages in the cache's order -> [pages, heads, token, dimension]"""
    return codes.view(-1, kh, 4, dp // 64, 4, 16, 16).permute(0, 1, 2, 5, 3, 4, 6).reshape(-1, kh, PAGE, dp)


def _value_values(codes, kh, dp):
    """value codes of pages in the cache's order -> [pages, heads, token, dimension]"""
    return codes.view(-1, kh, dp // 16, 4, 16, 4, 4).permute(0, 1, 5, 3, 6, 2, 4).reshape(-1, kh, PAGE, dp)


def _rows_at(counts, ends):
    """(sequence, position) of every row, for counts[i] rows that end at token ends[i] of their sequence"""
    n = torch.tensor(counts, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), n)
    first = torch.cumsum(n, 0) - n
    return seq, torch.arange(int(sum(counts)), device="cuda") - first[seq] + torch.tensor(ends, device="cuda")[seq] - n[seq]


def _places(dp):
    """where in a page's codes of one head the key and the value of (token, dimension) lie"""
    t, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(dp, device="cuda")[None, :]
    key = (((t // 16 * (dp // 64) + d // 64) * 4 + d % 64 // 16) * 16 + t % 16) * 16 + d % 16
    value = ((d // 16 * 4 + t % 16 // 4) * 16 + d % 16) * 16 + t // 16 * 4 + t % 4
    return key, value


def _plain_write(s):
    case = s["case"]
    kh, b, dim, dp = case["kv_heads"], case["block"], case["dim"], _row_dim(case["dim"])
    seq, pos = _rows_at(s["new"], s["kv_rows"])
    pages = s["pages"].to(torch.int64)
    page, slot = pages[seq, pos // PAGE], pos % PAGE
    per = PAGE // b
    begin = torch.tensor([t - n for n, t in zip(s["new"], s["kv_rows"])], device="cuda")  # the first new token of each sequence
    begin_page, begin_slot = pages[torch.arange(len(begin), device="cuda"), begin // PAGE], begin % PAGE
    going_on = begin_slot % b != 0  # the block that it falls into holds older tokens
    heads = torch.arange(kh, device="cuda")
    for x, codes, scale, place in ((s["k"], s["k_codes"], s["k_scale"], _places(dp)[0]), (s["v"], s["v_codes"], s["v_scale"], _places(dp)[1])):
        x = x.to(torch.float32)
        flat = scale.view(-1, kh, per)
        largest = torch.zeros(flat.shape[0] * per, kh, device="cuda")
        which = page * per + slot // b
        largest.scatter_reduce_(0, which[:, None].expand(-1, kh), x.abs().amax(-1), "amax")
        wanted = (largest * PER127).view(-1, per, kh).permute(0, 2, 1)
        old = flat[begin_page, :, begin_slot // b]  # [sequences, heads]
        floor = torch.where(going_on[:, None], old, torch.zeros_like(old))
        now = torch.maximum(wanted[begin_page, :, begin_slot // b], floor)
        touched = torch.zeros(flat.shape[0] * per, dtype=torch.bool, device="cuda")
        touched[which] = True
        fresh = torch.where(touched.view(-1, 1, per), wanted, flat)
        fresh[begin_page, :, begin_slot // b] = now
        # older tokens of a block whose scale grew: to the new scale
        factor = torch.where(now > 0, old / now, torch.zeros_like(old))
        token = begin_slot[:, None] // b * b + torch.arange(b, device="cuda")[None, :]  # [sequences, block]
        older = going_on[:, None] & (token < begin_slot[:, None])
        stored = codes.view(-1, kh, PAGE * dp)
        at = place[token][:, None]  # [sequences, 1, block, dp]
        who = begin_page[:, None, None, None]
        held = stored[who, heads[None, :, None, None], at]
        moved = ((held.to(torch.float32) - 128) * factor[:, :, None, None]).round().clamp(-127, 127)
        again = torch.where(older[:, None, :, None], (moved + 128).to(torch.uint8), held)
        stored[who, heads[None, :, None, None], at] = again
        # the new tokens
        mine = fresh[page, :, slot // b][:, :, None]
        q = torch.where(mine > 0, x / mine, torch.zeros_like(x)).round().clamp(-127, 127)
        stored[page[:, None, None], heads[None, :, None], place[slot][:, None, :dim]] = (q + 128).to(torch.uint8)
        flat.copy_(fresh)
    k, v = _plain_read(s)
    return k, v, s["k_scale"], s["v_scale"]


def _plain_read(s):
    case = s["case"]
    kh, b, dim, dp = case["kv_heads"], case["block"], case["dim"], _row_dim(case["dim"])
    seq, pos = _rows_at(s["back"], s["kv_rows"])
    page, slot = s["pages"].to(torch.int64)[seq, pos // PAGE], pos % PAGE
    k = _key_values(s["k_codes"], kh, dp)[page, :, slot, :dim].to(torch.float32).sub(128) * s["k_scale"][page, :, slot // b][:, :, None]
    v = _value_values(s["v_codes"], kh, dp)[page, :, slot, :dim].to(torch.float32).sub(128) * s["v_scale"][page, :, slot // b][:, :, None]
    return k.to(TYPES[case["type"]]), v.to(TYPES[case["type"]])


def _plain_attend(s):
    case = s["case"]
    kh, b, dim, dp, h = case["kv_heads"], case["block"], case["dim"], _row_dim(case["dim"]), case["heads"]
    seqs, table = s["pages"].shape
    group, longest, most = h // kh, table * PAGE, max(s["new"])
    pick = s["pages"].to(torch.int64).reshape(-1)

    def values(codes, scale, order):
        x = order(codes.view(-1, kh, PAGE * dp)[pick], kh, dp)[..., :dim].to(torch.float32) - 128
        x = x * scale[pick].repeat_interleave(b, -1)[..., None]
        return x.view(seqs, table, kh, PAGE, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kh, longest, dim)

    k = values(s["k_codes"], s["k_scale"], _key_values)
    seq, pos = _rows_at(s["new"], s["kv_rows"])
    ends = s["kv_len"].to(torch.int64)
    n = torch.tensor(s["new"], device="cuda")
    row = pos - (ends - n)[seq]
    q = torch.zeros(seqs, most, h, dim, device="cuda")
    q[seq, row] = s["q"].to(torch.float32)
    q = q.view(seqs, most, kh, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kh, most * group, dim)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    del k
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    score = score.view(seqs, kh, most, group, longest)
    at = (ends - n)[:, None] + torch.arange(most, device="cuda")[None, :]  # position of each row
    key = torch.arange(longest, device="cuda")
    seen = key[None, None, :] <= at[:, :, None]
    if case["window"]:
        seen &= key[None, None, :] > at[:, :, None] - case["window"]
    score = torch.where(seen[:, None, :, None, :], score, torch.full_like(score[:1, :1, :1, :1, :1], float("-inf")))
    top = score.amax(-1, keepdim=True)
    if case["sinks"]:
        sink = s["sinks"].view(1, kh, 1, group, 1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    del score
    total = p.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    out = torch.matmul(p.view(seqs, kh, most * group, longest), values(s["v_codes"], s["v_scale"], _value_values))
    out = out.view(seqs, kh, most, group, dim) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 2, 1, 3, 4).reshape(seqs, most, h, dim)[seq, row].to(TYPES[case["type"]])


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _token_index(dim, dp):
    """positions of token t's key and value in a page's codes of one head, written out token by token"""
    key = np.empty((PAGE, dim), np.int64)
    value = np.empty((PAGE, dim), np.int64)
    for t in range(PAGE):
        for d in range(dim):
            key[t, d] = 1024 * ((t >> 4) * (dp >> 6) + (d >> 6)) + 16 * (16 * ((d >> 4) & 3) + (t & 15)) + (d & 15)
            value[t, d] = 1024 * (d >> 4) + 16 * (16 * ((t >> 2) & 3) + (d & 15)) + 4 * (t >> 4) + (t & 3)
    return torch.from_numpy(key).cuda(), torch.from_numpy(value).cuda()


def _cached(s, i, count):
    """keys and values of the first `count` tokens of sequence i as [heads, tokens, dim] in 64 bits"""
    case = s["case"]
    kh, b, dim, dp = case["kv_heads"], case["block"], case["dim"], _row_dim(case["dim"])
    pages = s["pages"][i, : -(-count // PAGE)].long()
    got = []
    for codes, scale, index in zip((s["k_codes"], s["v_codes"]), (s["k_scale"], s["v_scale"]), _token_index(dim, dp)):
        c = codes.view(-1, kh, PAGE * dp)[pages][:, :, index.reshape(-1)].view(len(pages), kh, PAGE, dim).double() - 128
        c = c * scale[pages].double().repeat_interleave(b, 2)[..., None]
        got.append(c.transpose(0, 1).reshape(kh, -1, dim)[:, :count])
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return tuple(_exact_rope(s, s[n], s[n + "_weight"]) for n in ("q", "k"))
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "write":
        return _exact_write(s)
    both = [_cached(s, i, t) for i, t in enumerate(s["kv_rows"])]
    return tuple(torch.cat([b[j].transpose(0, 1) for b in both]) for j in (0, 1))


def _exact_rope(s, x, weight):
    case = s["case"]
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + 1e-6) * weight.double()
    spin = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None, None] * s["freqs"])
    part, rest = x[..., : case["rot"]], x[..., case["rot"]:]
    if case["pairs"] == "halves":
        a, b = part.chunk(2, -1)
        z = torch.complex(a, b) * spin
        return torch.cat([z.real, z.imag, rest], -1)
    z = torch.view_as_complex(part.reshape(*part.shape[:-1], -1, 2)) * spin
    return torch.cat([torch.view_as_real(z).flatten(-2), rest], -1)


def _exact_write(s):
    """A block's scale is the largest magnitude times 1/127, each in fp32, and never below the one its older tokens have;
    a code is the nearest whole number (ties to even) of the fp32 quotient."""
    case = s["case"]
    kh, b, dim, dp = case["kv_heads"], case["block"], case["dim"], _row_dim(case["dim"])
    back, scales = [], []
    for x, codes, scale, index in ((s["k"], s["k_codes"], s["k_scale"], 0), (s["v"], s["v_codes"], s["v_scale"], 1)):
        place = _token_index(dim, dp)[index]
        x, scale, stored, rows = x.double(), scale.double().clone(), codes.view(-1, kh, PAGE * dp), []
        row = 0
        for i, (n, t) in enumerate(zip(s["new"], s["kv_rows"])):
            for start in range((t - n) // b * b, t, b):
                page, blk = int(s["pages"][i, start // PAGE]), start % PAGE // b
                old = max(0, t - n - start)  # tokens of the block that were there
                end = min(start + b, t)
                mine = x[row: row + end - start - old]  # [tokens, heads, dim]
                row += end - start - old
                s0 = scale[page, :, blk] if old else torch.zeros(kh, dtype=torch.float64, device="cuda")
                s1 = torch.maximum((mine.abs().amax((0, 2)) * PER127).float().double(), s0)
                safe = torch.where(s1 > 0, s1, torch.ones_like(s1))
                q = (mine / safe[None, :, None]).float().double().round().clamp(-127, 127)
                slots = torch.arange(start % PAGE, start % PAGE + old, device="cuda")
                kept = stored[page][:, place[slots].reshape(-1)].view(kh, old, dim).transpose(0, 1).double() - 128
                kept = (kept * (s0 / safe).float().double()[None, :, None]).float().double().round().clamp(-127, 127)
                rows.append(torch.cat([kept, q]) * s1[None, :, None])
                scale[page, :, blk] = s1
        back.append(torch.cat(rows))
        scales.append(scale)
    return back[0], back[1], scales[0], scales[1]


def _exact_attend(s):
    case = s["case"]
    group, rows, out = case["heads"] // case["kv_heads"], 0, []
    for i, (n, t) in enumerate(zip(s["new"], s["kv_rows"])):
        k, v = _cached(s, i, t)
        q = s["q"][rows: rows + n].double()
        rows += n
        at = torch.arange(t - n, t, device="cuda")[:, None] - torch.arange(t, device="cuda")[None, :]
        hide = (at < 0) | (at >= case["window"]) if case["window"] else at < 0
        heads = []
        for h in range(case["heads"]):
            z = q[:, h] @ k[h // group].T * s["scale"]
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            z = z.masked_fill(hide, -math.inf)
            if case["sinks"]:
                z = torch.cat([z, s["sinks"][h].double().expand(n, 1)], 1)
            heads.append(torch.softmax(z, 1)[:, :t] @ v[h // group])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
