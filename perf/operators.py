"""The operators of the 4-bit paged KV cache: what is measured, and their plain forms.

The cache holds, for each layer, block and KV head, a K tile and a V tile of 1152
bytes: 16 rows (tokens) of 64 code bytes, then 16 rows of four fp16 parameters
(scale, minimum of dimensions 0-63; scale, minimum of dimensions 64-127).  A row's
32-bit word i holds dimensions 8i..8i+7: nibble j is dimension 8i + 2j, nibble 4 + j
dimension 8i + 2j + 1.  A code c stands for scale * c + minimum.

  write   quantise new K/V rows into the cache at their slots, then read back every
          row of the blocks they went to (the older rows beside them included)
  read    read rows of the cache back at their slots
  attend  causal varlen GQA attention of a step's query tokens (decodes of one token
          and prefill chunks) over the cache, in each of the case's layers
"""
import math
import random

import torch

own = False

HEAD_DIM, BLOCK, GROUP, HALF = 128, 16, 4, 64
CODE_BYTES, TILE_BYTES = BLOCK * HEAD_DIM // 2, BLOCK * HEAD_DIM // 2 + BLOCK * 8
LIMIT = 32768.0                     # rows are clamped to this range as they are written
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step's new rows of ten requests (the benchmark command's default): launch latency
        dict(name="write-decode-10", op="write", type="bf16", kv_heads=8, seqs=10, new=1, old=500, ragged=1),
        # a full prefill step: 16 chunks of 512 tokens, the engine's default token budget
        dict(name="write-prefill-8192", op="write", type="bf16", kv_heads=8, seqs=16, new=512, old=0, ragged=0),
        # the fp32 parity engine on the two-layer model's heads, ragged chunks that end inside blocks
        dict(name="write-fp32-odd", op="write", type="fp32", kv_heads=2, seqs=5, new=333, old=77, ragged=2),
        # a short request's rows handed to another consumer
        dict(name="read-short", op="read", type="bf16", kv_heads=8, tokens=100),
        # a whole request near the model's longest context
        dict(name="read-long", op="read", type="bf16", kv_heads=8, tokens=40001),
        # decode of the benchmark's ten requests, a few hundred tokens each
        dict(name="decode-10", op="attend", type="bf16", kv_heads=8, layers=4, decodes=10, decode_ctx=600,
             chunks=0, chunk=0, chunk_ctx=0, ragged=3),
        # a full decode batch of the serving benchmark
        dict(name="decode-256", op="attend", type="bf16", kv_heads=8, layers=1, decodes=256, decode_ctx=4096,
             chunks=0, chunk=0, chunk_ctx=0, ragged=4),
        # one request at the longest context: few rows, one long axis
        dict(name="decode-long", op="attend", type="bf16", kv_heads=8, layers=2, decodes=1, decode_ctx=40960,
             chunks=0, chunk=0, chunk_ctx=0, ragged=0),
        # one chunk late in a long prompt: fewer items than SMs
        dict(name="prefill-1x512", op="attend", type="bf16", kv_heads=8, layers=2, decodes=0, decode_ctx=0,
             chunks=1, chunk=512, chunk_ctx=3584, ragged=0),
        # a full prefill step, ragged chunks at different depths of their prompts
        dict(name="prefill-16x512", op="attend", type="bf16", kv_heads=8, layers=1, decodes=0, decode_ctx=0,
             chunks=16, chunk=512, chunk_ctx=7168, ragged=5),
        # continuous batching: prefill chunks beside running decodes
        dict(name="mixed-4-128", op="attend", type="bf16", kv_heads=8, layers=1, decodes=128, decode_ctx=2048,
             chunks=4, chunk=512, chunk_ctx=2048, ragged=6),
        # the fp32 parity engine on the two-layer model
        dict(name="fp32-mixed", op="attend", type="fp32", kv_heads=2, layers=2, decodes=5, decode_ctx=700,
             chunks=3, chunk=61, chunk_ctx=130, ragged=7),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    heads = rng.choice([1, 2, 4, 8])
    op = rng.choice(["write", "read", "attend", "attend", "attend"])
    ragged = rng.randrange(1, 1 << 20)
    if op == "write":
        seqs = _log_int(rng, 1, 64)
        return dict(op=op, type=kind, kv_heads=heads, seqs=seqs, new=_log_int(rng, 1, 8192 // seqs),
                    old=rng.randrange(0, 1000), ragged=ragged)
    if op == "read":
        return dict(op=op, type=kind, kv_heads=heads, tokens=_log_int(rng, 1, 40000))
    if kind == "fp32":              # the parity path: the small model's sizes
        return dict(op=op, type=kind, kv_heads=min(heads, 2), layers=2, decodes=rng.randrange(0, 8),
                    decode_ctx=_log_int(rng, 1, 1000), chunks=rng.randrange(1, 4), chunk=_log_int(rng, 2, 100),
                    chunk_ctx=rng.randrange(0, 300), ragged=ragged)
    shape = rng.choice(["decode", "decode", "prefill", "mixed"])
    decodes = 0 if shape == "prefill" else _log_int(rng, 1, 200)
    chunks = 0 if shape == "decode" else _log_int(rng, 1, 12)
    return dict(op=op, type=kind, kv_heads=heads, layers=rng.choice([1, 2]), decodes=decodes,
                decode_ctx=_log_int(rng, 1, min(40000, 400000 // max(1, decodes))), chunks=chunks,
                chunk=_log_int(rng, 2, 512), chunk_ctx=rng.randrange(0, 6000 // max(1, chunks)), ragged=ragged)


def _spread(rng, ragged, most, least):
    """A length up to `most`: that one, or for a ragged case anything down to a quarter of it."""
    return most if not ragged else rng.randint(max(least, most // 4), max(least, most))


def _write_lens(case):
    """(old rows, new rows) of each sequence."""
    rng = random.Random(case["ragged"])
    return [(rng.randint(0, case["old"]) if case["ragged"] else case["old"],
             _spread(rng, case["ragged"], case["new"], 1)) for _ in range(case["seqs"])]


def _attend_lens(case):
    """(query tokens, key tokens) of each sequence: the decodes, then the prefill chunks."""
    rng = random.Random(case["ragged"])
    lens = [(1, _spread(rng, case["ragged"], case["decode_ctx"], 1)) for _ in range(case["decodes"])]
    for _ in range(case["chunks"]):
        q = _spread(rng, case["ragged"], case["chunk"], 2)
        old = rng.randint(0, case["chunk_ctx"]) if case["ragged"] else case["chunk_ctx"]
        lens.append((q, old + q))
    return lens


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(shape, gen, dtype):
    """K or V rows as a layer produces them: near normal, a few stronger dimensions for each head, an offset."""
    gain = torch.rand(shape[-2:], generator=gen, device="cuda") * 0.6 + 0.7
    gain = torch.where(torch.rand(shape[-2:], generator=gen, device="cuda") < 0.03, 3 * gain, gain)
    bias = torch.randn(shape[-2:], generator=gen, device="cuda") * 0.3
    x = torch.randn(shape, generator=gen, device="cuda")
    return x.mul_(gain).add_(bias).to(dtype)


def _filled_cache(layers, blocks, heads, gen):
    """A cache whose every row was written before."""
    cache = torch.empty(layers, blocks, heads, 2, TILE_BYTES, dtype=torch.uint8, device="cuda")
    for layer in cache:
        for part in (0, 1):
            codes, params = _quantise(_rows((blocks, BLOCK, heads, HEAD_DIM), gen, torch.float32).transpose(1, 2))
            layer[:, :, part, :CODE_BYTES] = codes.flatten(-2)
            layer[:, :, part, CODE_BYTES:] = params.flatten(-2)
    return cache


def _block_rows(counts, gen, spare):
    """Block tables of sequences with `counts` blocks each, out of a shuffled pool, and the pool's size."""
    pool = sum(counts) + spare
    ids = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, pool


def _slots(table, seq, first, last):
    pos = torch.arange(first, last, device="cuda")
    return (table[seq].long()[pos // BLOCK] * BLOCK + pos % BLOCK).to(torch.int32)


def prepare(case, seed):
    gen, dtype, heads = _gen(seed), TYPES[case["type"]], case["kv_heads"]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["op"] == "read":
        n = case["tokens"]
        table, pool = _block_rows([-(-n // BLOCK)], gen, 9)
        return dict(case=case, cache=_filled_cache(1, pool, heads, gen), slots=_slots(table, 0, 0, n),
                    dtype=dtype, err=err)
    if case["op"] == "write":
        lens = _write_lens(case)
        table, pool = _block_rows([-(-(old + new) // BLOCK) for old, new in lens], gen, 9)
        tokens = sum(new for _, new in lens)
        # the rows as the QKV projection leaves them: V is a strided part of its output
        k = _rows((tokens, heads, HEAD_DIM), gen, dtype)
        qkv = torch.empty(tokens, (GROUP + 2) * heads * HEAD_DIM, dtype=dtype, device="cuda")
        qkv[:, -heads * HEAD_DIM:] = _rows((tokens, heads, HEAD_DIM), gen, dtype).flatten(1)
        v = qkv[:, -heads * HEAD_DIM:].unflatten(1, (heads, HEAD_DIM))
        slots = torch.cat([_slots(table, i, old, old + new) for i, (old, new) in enumerate(lens)])
        back = torch.cat([_slots(table, i, old // BLOCK * BLOCK, -(-(old + new) // BLOCK) * BLOCK)
                          for i, (old, new) in enumerate(lens)])
        return dict(case=case, cache=_filled_cache(1, pool, heads, gen), k=k, v=v, slots=slots, back=back,
                    dtype=dtype, err=err)
    lens = _attend_lens(case)
    table, pool = _block_rows([-(-kv // BLOCK) for _, kv in lens], gen, 9)
    tokens, layers = sum(q for q, _ in lens), case["layers"]
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor([q for q, _ in lens]), 0)
    q = (1.5 * torch.randn(layers, tokens, GROUP * heads, HEAD_DIM, generator=gen, device="cuda")).to(dtype)
    state = dict(case=case, cache=_filled_cache(layers, pool, heads, gen), q=q, out=torch.empty_like(q), table=table,
                 cu=cu.cuda(), kv=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda"),
                 seqs=len(lens), tokens=tokens, dtype=dtype, err=err)
    # the attention's workspace, as large as the engine's rule makes it: kept by the program
    state["workspace"] = torch.zeros(_workspace_bytes(len(lens), tokens, heads), dtype=torch.uint8, device="cuda")
    return state


def _workspace_bytes(seqs, tokens, heads):
    if own:
        from hayate_b200 import kernels as K
        return K.attention_workspace_size(seqs, tokens, heads)
    return 256


# ------------------------------------------------------------------ plain forms
def _quantise(x):
    """fp32 rows (..., 128) as code bytes (..., 64) and parameter bytes (..., 8)."""
    x = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (2, HALF))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    low, scale = lo.half(), ((hi - lo) * (1.0 / 15.0)).half()
    inverse = torch.ones_like(lo) / scale.float()
    code = torch.where(scale > 0, ((x - low.float()) * inverse).round().clamp(0, 15), 0).to(torch.uint8)
    code = code.flatten(-2).unflatten(-1, (HEAD_DIM // 8, 4, 2))          # word, pair j, which of the pair
    code = code.transpose(-1, -2).flatten(-2)                             # nibbles 0..7 of each word
    code = code.unflatten(-1, (4, 2))
    code = (code[..., 0] | (code[..., 1] << 4)).flatten(-2)               # bytes, low nibble first
    params = torch.stack([scale.squeeze(-1), low.squeeze(-1)], -1).flatten(-2).contiguous().view(torch.uint8)
    return code, params


def _values(codes, params):
    """fp32 rows (..., 128) of code bytes (..., 64) and parameter bytes (..., 8)."""
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (HEAD_DIM // 8, 2, 4))
    code = nib.transpose(-1, -2).flatten(-3).unflatten(-1, (2, HALF)).float()
    p = params.contiguous().view(torch.float16).float().unflatten(-1, (2, 2))
    return (code * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _parts(cache):
    """The cache's codes (..., heads, 2, 16, 64) and parameters (..., heads, 2, 16, 8), as views."""
    return cache[..., :CODE_BYTES].unflatten(-1, (BLOCK, HEAD_DIM // 2)), cache[..., CODE_BYTES:].unflatten(-1, (BLOCK, 8))


def _plain_read(cache, slots, dtype):
    codes, params = _parts(cache)
    blk, off = slots.long() // BLOCK, slots.long() % BLOCK
    x = _values(codes[blk, :, :, off], params[blk, :, :, off]).to(dtype)  # (tokens, heads, 2, 128)
    return x[:, :, 0].contiguous(), x[:, :, 1].contiguous()


def _plain_write(cache, k, v, slots):
    codes, params = _parts(cache)
    blk, off = slots.long() // BLOCK, slots.long() % BLOCK
    c, p = _quantise(torch.stack([k, v], 2))
    codes[blk, :, :, off] = c
    params[blk, :, :, off] = p


def _attend_padded(q, cache, table, lens_q, lens_k, scale):
    """Attention of one padded group: q (layers, seqs, rows, heads, 4, 128), key positions up to the table's width."""
    codes, params = _parts(cache)
    at = table.clamp(min=0).long()
    x = _values(codes[:, at], params[:, at])                              # (layers, seqs, blocks, heads, 2, 16, 128)
    x = x.permute(0, 1, 3, 4, 2, 5, 6).flatten(4, 5)                      # (layers, seqs, heads, 2, keys, 128)
    k, v = x[:, :, :, 0], x[:, :, :, 1]
    rows = q.shape[2]
    q = q.float().permute(0, 1, 3, 2, 4, 5).flatten(3, 4)                 # (layers, seqs, heads, rows * 4, 128)
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    last = (lens_k - lens_q)[:, None] + torch.arange(rows, device=q.device)
    last = torch.minimum(last, lens_k[:, None] - 1).repeat_interleave(GROUP, 1)
    hidden = torch.arange(k.shape[-2], device=q.device) > last[..., None]
    s = s.masked_fill_(hidden[None, :, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.unflatten(3, (rows, GROUP)).permute(0, 1, 3, 2, 4, 5)


def _plain_attend(s):
    """The decodes and the prefill chunks as two padded groups."""
    case, heads = s["case"], s["case"]["kv_heads"]
    out, scale = s["out"], 1.0 / math.sqrt(HEAD_DIM)
    q = s["q"].unflatten(2, (heads, GROUP))
    lens_q, lens_k, n = s["cu"][1:] - s["cu"][:-1], s["kv"], case["decodes"]
    if n:
        o = _attend_padded(q[:, :n, None], s["cache"], s["table"][:n, :-(-case["decode_ctx"] // BLOCK)],
                           lens_q[:n], lens_k[:n], scale)
        out[:, :n] = o[:, :, 0].flatten(2, 3).to(out.dtype)
    if case["chunks"]:
        j = torch.arange(case["chunk"], device="cuda")
        at = (s["cu"][n:-1, None] + j).clamp(max=s["tokens"] - 1).long()  # rows of each chunk, padded
        o = _attend_padded(q[:, at], s["cache"], s["table"][n:, :-(-(case["chunk_ctx"] + case["chunk"]) // BLOCK)],
                           lens_q[n:], lens_k[n:], scale)
        real = j < lens_q[n:, None]
        out[:, n:] = o[:, real].flatten(2, 3).to(out.dtype)
    return out


def run(s):
    op = s["case"]["op"]
    if own:
        from hayate_b200 import kernels as K
        if op == "write":
            K.kv_append_q4(s["k"], s["v"], s["slots"], s["cache"][0], err=s["err"])
            return K.kv_read_q4(s["cache"][0], s["back"], s["dtype"], err=s["err"])
        if op == "read":
            return K.kv_read_q4(s["cache"][0], s["slots"], s["dtype"], err=s["err"])
        K.attention_plan(s["cu"], s["kv"], s["seqs"], s["case"]["kv_heads"], s["seqs"], s["tokens"],
                         s["workspace"], s["err"])
        for layer in range(s["case"]["layers"]):
            K.varlen_attention_q4(s["q"][layer], s["out"][layer], s["cache"], layer, s["table"], s["cu"], s["kv"],
                                  s["seqs"], s["seqs"], s["tokens"], s["workspace"], err=s["err"])
        return s["out"]
    if op == "write":
        _plain_write(s["cache"][0], s["k"], s["v"], s["slots"])
        return _plain_read(s["cache"][0], s["back"], s["dtype"])
    if op == "read":
        return _plain_read(s["cache"][0], s["slots"], s["dtype"])
    return _plain_attend(s)


# ------------------------------------------------------------------ work
def work(case):
    size, heads = TYPES[case["type"]].itemsize, case["kv_heads"]
    wide, packed = 2 * heads * HEAD_DIM * size, 2 * heads * (HEAD_DIM // 2 + 8)   # a token's K and V
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (wide + packed + 4), "flops": case["tokens"] * heads * 4 * HEAD_DIM}
    if case["op"] == "write":
        lens = _write_lens(case)
        new = sum(n for _, n in lens)
        back = sum(-(-(o + n) // BLOCK) * BLOCK - o // BLOCK * BLOCK for o, n in lens)
        return {"bytes": (new + back) * (wide + packed + 4), "flops": heads * HEAD_DIM * (12 * new + 4 * back)}
    lens = _attend_lens(case)
    tokens, keys = sum(q for q, _ in lens), sum(kv for _, kv in lens)
    seen = sum(q * (kv - q) + q * (q + 1) // 2 for q, kv in lens)
    return {"bytes": case["layers"] * (keys * packed + 2 * tokens * GROUP * heads * HEAD_DIM * size),
            "flops": case["layers"] * 4 * HEAD_DIM * GROUP * heads * seen}


# ------------------------------------------------------------------ from the definition, in 64 bits
def _exact_rows(tile):
    """(..., 16, 128) values in 64 bits of tiles (..., 1152), nibble by nibble."""
    lead = tile.shape[:-1]
    codes = tile[..., :CODE_BYTES].reshape(*lead, BLOCK, HEAD_DIM // 2).to(torch.int64)
    par = tile[..., CODE_BYTES:].contiguous().view(torch.float16).reshape(*lead, BLOCK, 4).double()
    out = torch.empty(*lead, BLOCK, HEAD_DIM, dtype=torch.float64, device=tile.device)
    for nibble in range(8):
        byte, shift = nibble // 2, 4 * (nibble % 2)
        dim = 2 * nibble if nibble < 4 else 2 * (nibble - 4) + 1
        out[..., dim::8] = ((codes[..., byte::4] >> shift) & 15).double()
    out[..., :HALF] = out[..., :HALF] * par[..., 0:1] + par[..., 1:2]
    out[..., HALF:] = out[..., HALF:] * par[..., 2:3] + par[..., 3:4]
    return out


def _exact_quantised(x):
    """What rows x (tokens, heads, 128) stand for once written, group by group.  The codes' definition rounds to 32 bits
    at each step (difference, scale, inverse, quotient), so those roundings are made here too."""
    f32 = lambda t: t.float().double()  # noqa: E731
    got = []
    for g in (0, 1):
        y = x[..., HALF * g:HALF * (g + 1)].double().clamp(-LIMIT, LIMIT)
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        fifteenth = torch.tensor(1.0 / 15.0, dtype=torch.float32).double().item()
        m, s = lo.half().double(), f32(f32(hi - lo) * fifteenth).half().double()
        c = f32(f32(y - m) * f32(1.0 / torch.where(s > 0, s, 1.0))).round().clamp(0, 15)
        got.append(torch.where(s > 0, c, 0.0) * s + m)
    return torch.cat(got, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "attend":
        slots = (s["slots"] if case["op"] == "read" else s["back"]).long()
        tile = _exact_rows(s["cache"][0])                                 # (pool, heads, 2, 16, 128)
        if case["op"] == "write":
            new = s["slots"].long()
            for part, x in enumerate((s["k"], s["v"])):
                tile[new // BLOCK, :, part, new % BLOCK] = _exact_quantised(x)
        x = tile[slots // BLOCK, :, :, slots % BLOCK]
        return x[:, :, 0], x[:, :, 1]
    out, first = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (q_len, kv_len) in enumerate(_attend_lens(case)):
        blocks = s["table"][i, :-(-kv_len // BLOCK)].long()
        visible = torch.arange(kv_len, device="cuda") <= (kv_len - q_len + torch.arange(q_len, device="cuda"))[:, None]
        for layer in range(case["layers"]):
            x = _exact_rows(s["cache"][layer, blocks])                    # (blocks, heads, 2, 16, 128)
            x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :kv_len]
            for h in range(GROUP * case["kv_heads"]):
                z = s["q"][layer, first:first + q_len, h].double() @ x[h // GROUP, 0].T / math.sqrt(HEAD_DIM)
                out[layer, first:first + q_len, h] = torch.softmax(z.masked_fill(~visible, -math.inf), -1) @ x[h // GROUP, 1]
        first += q_len
    return out
