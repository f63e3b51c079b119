"""Operators for what sequences remember: linear attention by the gated delta rule, whose state is corrected token by token,
and the copies that branching sequences need: states of slots, blocks of a paged cache, forked and compacted block tables.

A case is one call, or a few as a server makes them together.  The plain forms work in 32 bits with elementary tensor
operations; exact() is the definition, token by token, in 64 bits.
"""
import ctypes as C
import math

import torch

own = False

CHUNK = 64   # tokens of a step of the plain form


# ------------------------------------------------------------------------------------------------ cases


def delta(name, type, prompts=0, portion=0, start=0, rows=0, ragged=False, qk_heads=16, heads=16, dim=64, vdim=64, norm=True, fused=False, samples=0):
    c = dict(op="delta", type=type, prompts=prompts, portion=portion, start=start, rows=rows, ragged=ragged, qk_heads=qk_heads, heads=heads,
             dim=dim, vdim=vdim, norm=norm, fused=fused, samples=samples)
    return dict(c, name=name) if name else c


def pool(name, op, type, layers, kv_heads, dim, blocks, **more):
    c = dict(op=op, type=type, layers=layers, kv_heads=kv_heads, dim=dim, blocks=blocks, **more)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's next token on a small fp32 model: the smallest call
        delta("delta-chat-f32", "f32", rows=1, qk_heads=4, heads=4),
        # a decoding batch of a large hybrid model: 64 users, value heads that share query and key heads
        delta("delta-decode-b64", "bf16", rows=64, qk_heads=16, heads=32, dim=128, vdim=128, fused=True),
        # a prompt of odd length in 32 bits, keys that come normed, as a replayed trace has it
        delta("delta-prompt-f32", "f32", prompts=1, portion=301, heads=16, qk_heads=16, norm=False),
        # continuous batching: prompt chunks of unlike lengths that continue, and users that already decode
        delta("delta-mixed", "bf16", prompts=3, portion=512, start=512, ragged=True, rows=11, qk_heads=32, heads=32, fused=True),
        # one prompt of 2K tokens
        delta("delta-prompt-2k", "bf16", prompts=1, portion=2048, qk_heads=16, heads=32, dim=128, vdim=128, fused=True),
        # a long document in one pass: the largest
        delta("delta-long", "bf16", prompts=1, portion=16384, qk_heads=8, heads=16, dim=128, vdim=128),
        # parallel samples of one prompt: its state goes to the samples' slots, and each takes a token of its own
        delta("states-samples-step", "bf16", rows=8, qk_heads=16, heads=32, dim=128, vdim=128, samples=8),
        # beams: states of all layers take the places that the last step chose
        dict(name="states-beams", op="states", layers=11, slots=40, slot_floats=32 * 64 * 64, beams=32),
        # eight samples of one prompt of 1,050 positions over fp16 pages of a 1.1B model: whole blocks are shared, the last one is copied
        pool("fork-samples", "fork", "f16", 22, 4, 64, 512, positions=1050, children=8),
        # a batch of beams over a pool in 32 bits: sixty-four branches
        pool("fork-wide-f32", "fork", "f32", 22, 4, 64, 512, positions=519, children=64),
        # half of a pool's users have left: what is in use moves to its front
        pool("compact-half", "compact", "f16", 22, 4, 64, 2048, live=0.5),
        # blocks of evicted users' prompts to their new places
        pool("copy-blocks-f32", "copy", "f32", 22, 4, 64, 768, pairs=256),
    ]


def draw(rng):
    """Another case of the ranges above."""
    def spread(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["decode", "decode", "prompt", "prompt", "prompt", "mixed", "samples", "states", "fork", "compact", "copy"])
    if kind in ("decode", "prompt", "mixed", "samples"):
        type = rng.choice(["bf16", "bf16", "f32"])
        qk = rng.choice([1, 2, 4, 8, 16])
        c = dict(type=type, qk_heads=qk, heads=qk * rng.choice([1, 1, 2, 3]), dim=rng.choice([32, 40, 64, 64, 96, 128, 128, 192, 256]),
                 vdim=rng.choice([32, 48, 64, 64, 100, 128, 128, 256]), norm=rng.random() < 0.7, fused=rng.random() < 0.5)
        most = max(2, 2 ** 25 // (c["heads"] * c["dim"] * c["vdim"]))   # 128 MB of states
        if kind == "decode":
            return delta(None, rows=min(most, spread(1, 64)), **c)
        if kind == "samples":
            n = min(most, spread(2, 16))
            return delta(None, rows=n, samples=n, **c)
        prompts, longest = rng.choice([1, 1, 2, 4]), 8192 if type == "bf16" else 1024
        portion = spread(2, longest // prompts // (4 if c["dim"] > 128 or c["heads"] > 16 else 1))
        return delta(None, prompts=prompts, portion=portion, start=rng.choice([0, 0, portion]), ragged=rng.random() < 0.5, rows=min(most, spread(1, 24)) if kind == "mixed" else 0, **c)
    if kind == "states":
        slots = spread(4, 48)
        return dict(op="states", layers=spread(1, min(16, 440 // slots)), slots=slots, slot_floats=rng.choice([4 * 64 * 64, 16 * 64 * 64, 32 * 64 * 64, 5 * 40 * 100, 7 * 3 * 515]),
                    beams=rng.randint(2, slots))
    type = rng.choice(["f16", "f32"])
    c = dict(type=type, layers=spread(2, 22), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([48, 64, 64, 96]))
    if kind == "fork":
        return pool(None, "fork", blocks=256, positions=spread(1, 3000), children=spread(1, 64), **c)
    most = 2 ** 28 // (c["layers"] * 16 * c["kv_heads"] * c["dim"] * (2 if type == "f16" else 4))   # a quarter of a GB each for keys and values
    if kind == "compact":
        return pool(None, "compact", blocks=min(most, spread(64, 1500)), live=rng.choice([0.2, 0.5, 0.8]), **c)
    blocks = min(most, spread(32, 700))
    return pool(None, "copy", blocks=blocks, pairs=rng.randint(1, blocks // 3), **c)


def spans(c):
    """(cached positions, new tokens) of each sequence of a batch."""
    out = []
    for i in range(c["prompts"]):
        n = c["portion"] if not c["ragged"] else max(2, round(c["portion"] * (1.0 - 0.6 * ((i * 0.6180339887) % 1.0))))
        out.append((c["start"], n))
    return out + [(100 + 7 * i, 1) for i in range(c["rows"])]


# ------------------------------------------------------------------------------------------------ what a program has in hand

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    pick = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    c = case
    if c["op"] == "states":
        n, slots = c["beams"], c["slots"]
        state = normal(c["layers"], slots, c["slot_floats"])
        to = torch.randperm(slots, generator=pick)[:n]
        start = to[torch.randint(0, n, (n,), generator=pick)]   # every beam's parent is one of the beams
        return dict(case=c, state=state, frm=start.tolist(), to=to.tolist())
    if c["op"] == "delta":
        T, Q, H, d, e = sum(n for _, n in spans(c)), c["qk_heads"], c["heads"], c["dim"], c["vdim"]
        width = 2 * Q * d + H * e
        rows = normal(T, width)
        if not c["norm"]:   # keys come normed, queries too
            qk = rows[:, :2 * Q * d].view(T, 2 * Q, d)
            qk /= qk.square().sum(-1, keepdim=True).add(1e-6).sqrt()
        rows = rows.to(TYPES[c["type"]])
        q, k, v = rows.split([Q * d, Q * d, H * e], 1)
        if not c["fused"]:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        # slow and fast heads, tokens that erase more and less
        rate = torch.exp(torch.empty(H, device="cuda").uniform_(math.log(0.003), math.log(1.5), generator=gen))
        g = -rate * torch.nn.functional.softplus(normal(T, H))
        beta = torch.sigmoid(normal(T, H))
        N = len(spans(c))
        slots = N + 3
        at = torch.randperm(slots, generator=pick)[:N].tolist()
        state = 0.3 * normal(slots, H, d, e)
        s = dict(case=c, q=q, k=k, v=v, g=g, beta=beta, state=state, slots=at, out=torch.empty((T, H, e), device="cuda", dtype=rows.dtype),
                 frm=[], to=[], scale=d ** -0.5)
        if c["samples"]:
            parent = next(i for i in range(slots) if i not in at)
            s["frm"], s["to"] = [parent] * c["samples"], at
        return s
    shape = (c["layers"], c["blocks"], 16, c["kv_heads"], c["dim"])
    s = dict(case=c, k=normal(*shape).to(TYPES[c["type"]]), v=normal(*shape).to(TYPES[c["type"]]))
    order = torch.randperm(c["blocks"], generator=pick).tolist()
    if c["op"] == "copy":
        s["frm"], s["to"] = order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]
    elif c["op"] == "fork":
        n = -(-c["positions"] // 16)
        s["table"], s["free"] = order[:n], order[n:]
    else:
        n = max(1, round(c["blocks"] * c["live"]))
        cuts = sorted({0, n, *torch.randint(0, n, (min(31, n),), generator=pick).tolist()})
        s["tables"], s["free"] = [order[a:b] for a, b in zip(cuts, cuts[1:])], order[n:]
    return s


def work(case):
    c = case
    if c["op"] == "states":
        return dict(bytes=2 * 4 * c["layers"] * c["beams"] * c["slot_floats"], flops=0)
    if c["op"] == "delta":
        size, H, S = 2 if c["type"] == "bf16" else 4, c["heads"], 4 * c["heads"] * c["dim"] * c["vdim"]
        T = sum(n for _, n in spans(c))
        states = sum(S + (S if cached else 0) for cached, _ in spans(c))
        if c["samples"]:
            states = S + c["samples"] * S   # the parent's read, the samples' written
        return dict(bytes=states + T * (size * (2 * c["qk_heads"] * c["dim"] + 2 * H * c["vdim"]) + 8 * H), flops=6.0 * T * H * c["dim"] * c["vdim"])
    block = 2 * c["layers"] * 16 * c["kv_heads"] * c["dim"] * (2 if c["type"] == "f16" else 4)
    if c["op"] == "copy":
        return dict(bytes=2 * c["pairs"] * block, flops=0)
    if c["op"] == "fork":
        tail = c["positions"] % 16 != 0
        return dict(bytes=(1 + c["children"]) * block if tail else 4 * c["children"] * (c["positions"] // 16), flops=0)
    live = max(1, round(c["blocks"] * c["live"]))
    return dict(bytes=2 * max(1.0, live * (1 - c["live"])) * block, flops=0)


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits


def unit(x, c):
    """Queries or keys of a batch [tokens, heads, dim] for every value head."""
    x = x.float().unflatten(1, (c["qk_heads"], c["dim"]))
    if c["norm"]:
        x = x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    return x.repeat_interleave(c["heads"] // c["qk_heads"], 1)


def inverse(A):
    """(I + A)^-1 for strictly lower triangular A [..., n, n], n a power of two: blocks of one, two, four ..."""
    n = A.shape[-1]
    T = torch.eye(n, device=A.device, dtype=A.dtype).expand(A.shape).clone()
    b = 1
    while b < n:
        blocks = T.unflatten(-1, (n // (2 * b), 2 * b)).unflatten(-3, (n // (2 * b), 2 * b))
        at = torch.arange(n // (2 * b), device=A.device)
        mine = blocks[..., at, :, at, :]                      # [block, ..., 2b, 2b]
        low = A.unflatten(-1, (n // (2 * b), 2 * b)).unflatten(-3, (n // (2 * b), 2 * b))[..., at, :, at, :][..., b:, :b]
        mine[..., b:, :b] = -(mine[..., b:, b:].contiguous() @ low.contiguous() @ mine[..., :b, :b].contiguous())
        blocks[..., at, :, at, :] = mine
        b *= 2
    return T


def one_token(s, q, k, v, g, beta, slots):
    S = s["state"][slots] * g.exp()[..., None, None]
    u = beta[..., None] * (v - (k[..., None] * S).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    s["state"][slots] = S
    return s["scale"] * (q[..., None] * S).sum(-2)


def portions(s, q, k, v, g, beta, slots, fresh):
    """[sequences, heads, chunks, CHUNK, ...]: chunk by chunk, all sequences and heads together."""
    G = g.double().cumsum(-1)
    fade = (G[..., :, None] - G[..., None, :]).float()
    low = torch.ones(CHUNK, CHUNK, device=g.device, dtype=torch.bool).tril()
    fade = torch.where(low, fade, -math.inf).exp()
    kt = k.transpose(-1, -2).contiguous()
    A = (beta[..., None] * fade * (k @ kt)).tril(-1)
    T = inverse(A) * beta[..., None, :]
    P = fade * (q @ kt)
    first, last = G.float().exp()[..., None], (G[..., -1:] - G).float().exp()[..., None]
    S = s["state"][slots] * ~fresh[:, None, None, None]
    out = torch.empty_like(v)
    for i in range(k.shape[2]):
        u = T[:, :, i] @ (v[:, :, i] - first[:, :, i] * (k[:, :, i] @ S))
        out[:, :, i] = first[:, :, i] * (q[:, :, i] @ S) + P[:, :, i] @ u
        S = first[:, :, i, -1:] * S + kt[:, :, i] @ (last[:, :, i] * u)
    s["state"][slots] = S
    return s["scale"] * out


def plain_delta(s):
    c = s["case"]
    if s["to"]:
        s["state"][s["to"]] = s["state"][s["frm"]]
    q, k, v = unit(s["q"], c), unit(s["k"], c), s["v"].float().unflatten(1, (c["heads"], c["vdim"]))
    out, seqs = s["out"], spans(c)
    many, first = c["prompts"], sum(n for _, n in seqs[:c["prompts"]])
    if many:
        lengths = torch.tensor([n for _, n in seqs[:many]], device="cuda")
        longest = -(-max(n for _, n in seqs[:many]) // CHUNK) * CHUNK
        at = torch.arange(longest, device="cuda")
        inside = at < lengths[:, None]                                   # [sequences, tokens]
        token = torch.where(inside, at + (lengths.cumsum(0) - lengths)[:, None], 0)

        def chunks(x):   # -> [sequences, heads, chunks, CHUNK, ...], zeros behind the last token
            x = x[token] * inside.view(*inside.shape, *([1] * (x.dim() - 1)))
            return x.transpose(1, 2).unflatten(2, (longest // CHUNK, CHUNK)).contiguous()

        fresh = torch.tensor([cached == 0 for cached, _ in seqs[:many]], device="cuda")
        o = portions(s, chunks(q), chunks(k), chunks(v), chunks(s["g"]), chunks(s["beta"]), s["slots"][:many], fresh)
        out[:first] = o.flatten(2, 3).transpose(1, 2)[inside].to(out.dtype)
    if c["rows"]:
        out[first:] = one_token(s, q[first:], k[first:], v[first:], s["g"][first:], s["beta"][first:], s["slots"][many:]).to(out.dtype)
    return dict(out=out, state=s["state"])


def plain_states(s):
    s["state"][:, s["to"]] = s["state"][:, s["frm"]]
    return s["state"]


def moves(s):
    """Blocks in use, in the order of their numbers, to the lowest numbers: (from, to), the new tables, the free stack."""
    used = sorted(b for t in s["tables"] for b in t)
    high, holes = [b for b in used if b >= len(used)], sorted(set(range(len(used))) - set(used))
    place = dict(zip(high, holes))
    return high, holes, [[place.get(b, b) for b in t] for t in s["tables"]], list(range(s["case"]["blocks"] - 1, len(used) - 1, -1))


def plain_pool(s):
    c = s["case"]
    if c["op"] == "copy":
        frm, to, more = s["frm"], s["to"], {}
    elif c["op"] == "fork":
        whole, tail = c["positions"] // 16, c["positions"] % 16 != 0
        to = s["free"][::-1][:c["children"]] if tail else []
        frm = s["table"][whole:] * len(to)
        more = dict(tables=torch.tensor([s["table"][:whole] + to[i:i + 1] for i in range(c["children"])]))
    else:
        frm, to, tables, free = moves(s)
        more = dict(tables=torch.tensor([b for t in tables for b in t]), free=torch.tensor(free))
    if to:
        for x in (s["k"], s["v"]):
            x[:, to] = x[:, frm]
    return dict(k=s["k"], v=s["v"], **more)


# ------------------------------------------------------------------------------------------------ the library's calls

LIB = None


def library():
    global LIB
    if LIB is None:
        from nvllm_amd import capi
        LIB = capi.load_hip()
        LIB.init_ops()
    return LIB


def ints(values):
    return (C.c_int * max(1, len(values)))(*values)


def table(capi, blocks, room):
    at = (C.c_int * max(1, room))(*blocks)
    t = capi.BlockTable(C.cast(at, C.POINTER(C.c_int)), len(blocks))
    return t, at


def handles(s):
    """What a server keeps for its batch or its pool: made on the first pass."""
    if "args" in s:
        return s["args"]
    from nvllm_amd import capi
    lib, c = library(), s["case"]
    if c["op"] in ("states", "delta"):
        a = dict(frm=ints(s["frm"]), to=ints(s["to"]))
        if c["op"] == "delta":
            seqs = list(zip(s["slots"], spans(c)))
            a["ids"] = ints([slot for slot, (_, n) in seqs for _ in range(n)])
            a["pos"] = ints([cached + i for _, (cached, n) in seqs for i in range(n)])
    else:
        m = capi.KVCacheManager()
        size = s["k"].element_size()
        if lib.nvllm_attach_kv_pool(C.byref(m), 16, c["blocks"], c["layers"], c["kv_heads"], c["dim"], size, s["k"].data_ptr(), s["v"].data_ptr()):
            raise RuntimeError("nvllm_attach_kv_pool")
        a = dict(manager=m)
        if c["op"] == "copy":
            a.update(frm=ints(s["frm"]), to=ints(s["to"]))
        else:
            tables = [s["table"]] if c["op"] == "fork" else s["tables"]
            a["first"] = [table(capi, t, len(t)) for t in tables]
            a["free"] = ints(s["free"])
            C.memmove(m.free_block_indices, a["free"], 4 * len(s["free"]))
            m.free_blocks_count = len(s["free"])
            records = [table(capi, [], len(s["table"])) for _ in range(c["children"])] if c["op"] == "fork" else [table(capi, t, len(t)) for t in tables]
            a["records"] = records
            a["tables"] = (C.POINTER(capi.BlockTable) * len(records))(*[C.pointer(t) for t, _ in records])
    s["args"] = a
    return a


def done(status):
    if status < 0:
        raise RuntimeError("the library refused the call: %d" % status)


def own_delta(s):
    lib, c, a = library(), s["case"], handles(s)
    slots, H, d, e = s["state"].shape
    if s["to"]:
        done(lib.nvllm_copy_states(s["state"].data_ptr(), 4 * H * d * e, 1, slots, a["frm"], a["to"], len(s["to"])))
    q, k, v, out = s["q"], s["k"], s["v"], s["out"]
    done(lib.nvllm_gated_delta(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), s["g"].data_ptr(), s["beta"].data_ptr(), s["state"].data_ptr(), a["ids"], a["pos"],
                               slots, s["scale"], 1e-6 if c["norm"] else 0.0, c["qk_heads"], H, d, e, q.stride(0), k.stride(0), v.stride(0), q.element_size(), len(q)))
    return dict(out=out, state=s["state"])


def own_states(s):
    lib, a = library(), handles(s)
    state = s["state"]
    done(lib.nvllm_copy_states(state.data_ptr(), 4 * state.shape[2], state.shape[0], state.shape[1], a["frm"], a["to"], len(s["to"])))
    return state


def own_pool(s):
    lib, c, a = library(), s["case"], handles(s)
    m = C.byref(a["manager"])
    more = {}
    if c["op"] == "copy":
        done(lib.nvllm_copy_blocks(m, a["frm"], a["to"], len(s["to"])))
    elif c["op"] == "fork":
        n = c["children"]
        done(lib.nvllm_fork_tables(m, C.byref(a["first"][0][0]), c["positions"], a["tables"], n))
        more["tables"] = torch.tensor([at[:t.num_blocks] for t, at in a["records"]])
        for t, _ in reversed(a["records"]):   # the samples end: the pool is as it was
            done(lib.nvllm_free_table(m, C.byref(t)))
    else:
        for (_, at), (_, first) in zip(a["records"], a["first"]):
            C.memmove(at, first, C.sizeof(first))
        C.memmove(a["manager"].free_block_indices, a["free"], 4 * len(s["free"]))
        done(lib.nvllm_compact_blocks(m, a["tables"], len(a["records"])))
        more["tables"] = torch.tensor([b for t, at in a["records"] for b in at[:t.num_blocks]])
        more["free"] = torch.tensor(a["manager"].free_block_indices[:a["manager"].free_blocks_count])
    return dict(k=s["k"], v=s["v"], **more)


def run(state):
    op = state["case"]["op"]
    if own:
        return own_delta(state) if op == "delta" else own_states(state) if op == "states" else own_pool(state)
    return plain_delta(state) if op == "delta" else plain_states(state) if op == "states" else plain_pool(state)


# ------------------------------------------------------------------------------------------------ the definition, 64 bits


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "states":
        return torch.stack([s["state"][:, s["frm"][s["to"].index(i)] if i in s["to"] else i] for i in range(c["slots"])], 1).double()
    if c["op"] == "delta":
        H, Q, d = c["heads"], c["qk_heads"], c["dim"]
        state = s["state"].double()
        for f, t in zip(s["frm"], s["to"]):
            state[t] = s["state"][f].double()
        share = torch.arange(H, device="cuda") // (H // Q)
        q, k, v = s["q"].double().view(-1, Q, d)[:, share], s["k"].double().view(-1, Q, d)[:, share], s["v"].double().view(-1, H, c["vdim"])
        if c["norm"]:
            q, k = (x * torch.rsqrt(torch.linalg.vecdot(x, x) + 1e-6)[..., None] for x in (q, k))
        decay, beta = torch.exp(s["g"].double()), s["beta"].double()
        out = torch.zeros(len(q), H, c["vdim"], device="cuda", dtype=torch.float64)
        seqs, at = spans(c), 0
        starts = []
        for (cached, n), slot in zip(seqs, s["slots"]):
            starts.append(at)
            at += n
            if cached == 0:
                state[slot] = 0.0
        # sequences side by side, the longest first: at step i those that have a token i
        order = sorted(range(len(seqs)), key=lambda j: -seqs[j][1])
        slots, where = torch.tensor([s["slots"][j] for j in order], device="cuda"), torch.tensor([starts[j] for j in order], device="cuda")
        lengths = [seqs[j][1] for j in order]
        S, live = state[slots], len(order)
        for i in range(lengths[0]):
            while lengths[live - 1] <= i:
                live -= 1
            t, M = where[:live] + i, S[:live]
            M.mul_(decay[t, :, None, None])
            M.add_(k[t].unsqueeze(-1) * (beta[t, :, None] * (v[t] - torch.matmul(k[t].unsqueeze(-2), M).squeeze(-2))).unsqueeze(-2))
            out[t] = torch.matmul(q[t].unsqueeze(-2), M).squeeze(-2) * s["scale"]
        state[slots] = S
        return dict(out=out, state=state)
    frm, to, more = s.get("frm"), s.get("to"), {}
    if c["op"] == "fork":
        keep, n = c["positions"] // 16, c["children"]
        to = [s["free"][-1 - i] for i in range(n)] if c["positions"] % 16 else []
        frm, more = [s["table"][-1]] * len(to), dict(tables=None)
    elif c["op"] == "compact":
        used = sorted(sum(s["tables"], []))
        frm, to, more = [b for b in used if b >= len(used)], [b for b in range(len(used)) if b not in set(used)], dict(tables=None, free=None)
    source = torch.arange(c["blocks"], device="cuda")
    source[torch.tensor(to, device="cuda", dtype=torch.long)] = torch.tensor(frm, device="cuda", dtype=torch.long)
    return dict(k=s["k"].double()[:, source], v=s["v"].double()[:, source], **more)
