"""The serving step's operators over a paged latent cache, as cases to measure.

Four operators a batch of requests goes through at each step of a latent-attention (MLA) model:

  plan    block tables, cache rows (slots), positions and ancestor masks of the step's new tokens, from
          request lengths and the tree of drafted tokens
  rows    the new tokens' latents: rmsnorm, rotary pairs, rounding to the cache's type, stored at their slots
  attn    attention of every new token over its request's cached rows and its own branch of the tree
  logits  penalties for repeated tokens, biases and grammar masks on the rows of logits that follow

Sizes are the ones this repository is configured and benchmarked with (32 heads, latents of 512 + 64, 4096
positions, a vocabulary of 163840, batches of 1, 16 and 64) and generic ones around them. Request lengths
are ragged and follow from the case alone; the seed makes the values.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
NEG = float("-inf")


# ---- the cases ----------------------------------------------------------------------------------------

def listed():
    return [
        # one new token for each of 64 requests: what every decode step of a full batch begins with
        {"name": "plan_decode_64", "op": "plan", "B": 64, "ctx": 4096, "q": 1, "page": 64, "tree": False},
        # 256 requests with trees of up to 31 drafted tokens, small pages, long tables, a pool that runs short
        {"name": "plan_tree_256", "op": "plan", "B": 256, "ctx": 32768, "q": 31, "page": 16, "tree": True},
        # a decode batch's latents without rotary pairs (the Kimi-Linear form)
        {"name": "rows_bf16_64", "op": "rows", "T": 64, "kl": 512, "rope": 64, "nope": True, "dtype": "bf16"},
        # a prompt chunk's latents with rotary pairs at far positions
        {"name": "rows_f16_8191", "op": "rows", "T": 8191, "kl": 512, "rope": 64, "nope": False, "dtype": "f16"},
        # the engine's own decode: one token over 4096 cached fp32 rows
        {"name": "attn_f32_1x4096", "op": "attn", "B": 1, "ctx": 4095, "q": 1, "heads": 32, "kl": 512,
         "rope": 64, "page": 64, "tree": False, "dtype": "f32"},
        # a decode batch of 64 at up to 4096 positions: bound by the cache's bytes
        {"name": "attn_bf16_decode_64", "op": "attn", "B": 64, "ctx": 4095, "q": 1, "heads": 32, "kl": 512,
         "rope": 64, "page": 64, "tree": False, "dtype": "bf16"},
        # 16 requests checking trees of up to 16 drafted tokens
        {"name": "attn_bf16_tree_16", "op": "attn", "B": 16, "ctx": 4099, "q": 16, "heads": 32, "kl": 512,
         "rope": 64, "page": 32, "tree": True, "dtype": "bf16"},
        # two long contexts with small trees: few rows, so the length has to be split
        {"name": "attn_f16_long_2", "op": "attn", "B": 2, "ctx": 131003, "q": 5, "heads": 32, "kl": 512,
         "rope": 64, "page": 16, "tree": True, "dtype": "f16"},
        # a prompt's chunk of 512 tokens behind 8192 cached ones: bound by the matrix products
        {"name": "attn_bf16_chunk_512", "op": "attn", "B": 1, "ctx": 8192, "q": 512, "heads": 32, "kl": 512,
         "rope": 64, "page": 64, "tree": False, "dtype": "bf16"},
        # one row of logits, every adjustment
        {"name": "logits_f32_1", "op": "logits", "B": 1, "q": 1, "V": 163840, "hist": 4096, "bias": 64,
         "dtype": "f32"},
        # a decode batch of 64 with 16-bit logits
        {"name": "logits_bf16_64", "op": "logits", "B": 64, "q": 1, "V": 163840, "hist": 4096, "bias": 300,
         "dtype": "bf16"},
        # the rows of 16 trees of up to 16 drafted tokens, each with its own branch's tokens counted
        {"name": "logits_f32_tree_16", "op": "logits", "B": 16, "q": 16, "V": 163840, "hist": 8192, "bias": 64,
         "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rows", "attn", "attn", "logits"])
    if op == "plan":
        B, tree = _log(rng, 1, 512), rng.random() < 0.5
        return {"op": op, "B": B, "ctx": _log(rng, 1, 32768), "q": _log(rng, 1, 31 if tree else 64),
                "page": rng.choice([1, 16, 24, 32, 64, 128]), "tree": tree}
    if op == "rows":
        kl, rope = rng.choice([(512, 64), (512, 64), (256, 32), (64, 16), (500, 62)])
        return {"op": op, "T": _log(rng, 1, 8191), "kl": kl, "rope": rope, "nope": rng.random() < 0.3,
                "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op == "attn":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        kl, rope = rng.choice([(512, 64), (512, 64), (512, 64), (256, 32), (128, 16), (64, 16)])
        tree = rng.random() < 0.5
        c = {"op": op, "B": _log(rng, 1, 64), "ctx": _log(rng, 1, 60000), "q": _log(rng, 1, 64),
             "heads": rng.choice([4, 16, 20, 32, 32, 64]), "kl": kl, "rope": rope,
             "page": rng.choice([1, 16, 24, 32, 64, 64, 128]), "tree": tree, "dtype": dtype}
        # no more than the largest listed cases: rows of cache, and products
        while c["B"] * (c["ctx"] + c["q"]) > 262144 or \
                c["B"] * c["q"] * c["heads"] * (c["ctx"] + c["q"]) > (2 ** 26 if dtype != "f32" else 2 ** 24):
            c["ctx" if c["ctx"] > 64 and rng.random() < 0.6 else "q" if c["q"] > 1 else "B" if c["B"] > 1 else "ctx"] //= 2
        c["ctx"], c["q"], c["B"] = max(1, c["ctx"]), max(1, c["q"]), max(1, c["B"])
        return c
    B = _log(rng, 1, 64)
    return {"op": op, "B": B, "q": _log(rng, 1, max(1, 256 // B)), "V": _log(rng, 1000, 163840),
            "hist": _log(rng, 1, 8192), "bias": _log(rng, 1, 300), "dtype": rng.choice(["f32", "f16", "bf16"])}


# ---- inputs --------------------------------------------------------------------------------------------

def _lens(B, most, ragged=0.6):
    """B lengths up to `most` (the first is `most` itself), the same for a case every time."""
    return [max(1, int(round(most * (1.0 - ragged * ((r * 0.6180339887) % 1.0))))) for r in range(B)]


def _qlens(case):
    return _lens(case["B"], case["q"], 0.6 if case.get("tree") or case["op"] == "logits" else 0.0)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _indptr(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _parents(rng, qlens):
    """Trees as a drafter makes them: a spine with branches; a parent is an earlier node, or -1 at a root."""
    out = []
    for n in qlens:
        out += [-1 if i == 0 else (i - 1 if rng.random() < 0.5 else rng.randrange(-1 if rng.random() < 0.1 else 0, i))
                for i in range(n)]
    return out


def _mask_words(parents, qlens, words):
    """Each node's ancestors and itself as bits, in signed 32-bit words."""
    rows, at = [], 0
    for n in qlens:
        bits = []
        for i in range(n):
            p = parents[at + i]
            bits.append((bits[p] if p >= 0 else 0) | (1 << i))
        for b in bits:
            ws = [(b >> (32 * w)) & 0xFFFFFFFF for w in range(words)]
            rows.append([w - (1 << 32) if w >= 1 << 31 else w for w in ws])
        at += n
    return rows


def _padded(ctx, page):
    return -(-ctx // page)


def prepare(case, seed):
    st = {"case": case}
    rng, g = random.Random(seed), _gen(seed)
    op = case["op"]
    if op == "rows":
        T, kl, rope = case["T"], case["kl"], case["rope"]
        n = T + 61
        st["x"] = torch.randn(T, kl + rope, generator=g, device="cuda") * 1.7
        st["w"] = 1.0 + 0.2 * torch.randn(kl, generator=g, device="cuda")
        st["inv_freq"] = 10000.0 ** (-torch.arange(0, rope, 2, device="cuda", dtype=torch.float32) / rope)
        st["pos"] = torch.randint(0, 1 << 20, (T,), generator=g, device="cuda", dtype=torch.int32)
        st["slot"] = torch.randperm(n, generator=g, device="cuda")[:T].contiguous()
        st["cache"] = torch.randn(n, kl + rope, generator=g, device="cuda").to(DTYPES[case["dtype"]])
    elif op == "plan":
        B, page = case["B"], case["page"]
        ctx, q = _lens(B, case["ctx"]), _qlens(case)
        T = sum(q)
        held = [_padded(c, page) + (1 if rng.random() < 0.2 else 0) for c in ctx]
        need = [max(0, _padded(c + n, page) - h) for c, n, h in zip(ctx, q, held)]
        cols = max(_padded(c + n, page) for c, n in zip(ctx, q)) + 1
        pool = sum(held) + sum(need) + 8
        ids = list(range(pool))
        rng.shuffle(ids)
        table, at = [], 0
        for h in held:
            table.append(ids[at:at + h] + [-1] * (cols - h))
            at += h
        free = ids[at:]
        # the pool of the larger listed batch is a little short: the last requests go without
        n_free = max(1, sum(need) - 3) if case["tree"] and sum(need) > 3 else len(free)
        st.update(ctx_len=_ints(ctx), q_len=_ints(q), held=_ints(held), table=_ints(table),
                  free=_ints(free[:n_free]), head=_ints([0]), T=T, Q=max(q), words=-(-max(q) // 32))
        st["parent"] = _ints(_parents(rng, q)) if case["tree"] else None
        st.update(held_out=torch.zeros(B, dtype=torch.int32, device="cuda"),
                  head_out=_ints([0]), q_indptr=torch.zeros(B + 1, dtype=torch.int32, device="cuda"),
                  kv_len=torch.zeros(B, dtype=torch.int32, device="cuda"),
                  pos=torch.zeros(T, dtype=torch.int32, device="cuda"),
                  slot=torch.zeros(T, dtype=torch.int64, device="cuda"),
                  mask=torch.zeros(T, st["words"], dtype=torch.int32, device="cuda"), short=_ints([0]))
    elif op == "attn":
        B, page, H, kl, rope = case["B"], case["page"], case["heads"], case["kl"], case["rope"]
        dt, D = DTYPES[case["dtype"]], case["kl"] + case["rope"]
        q = _qlens(case)
        kv = [c + n for c, n in zip(_lens(B, case["ctx"]), q)]
        blocks = [_padded(k, page) for k in kv]
        cols, pool = max(blocks), sum(blocks) + 3
        ids = torch.randperm(pool, generator=g, device="cuda", dtype=torch.int32)
        col = torch.arange(cols, device="cuda")[None, :]
        start = _ints(_indptr(blocks)[:-1])[:, None]
        st["table"] = torch.where(col < _ints(blocks)[:, None], ids[(start + col).clamp(max=pool - 1)], -1) \
            .to(torch.int32).contiguous()
        T, words = sum(q), -(-max(q) // 32)
        st["q"] = torch.randn(T, H, D, generator=g, device="cuda").to(dt)
        st["cache"] = torch.randn(pool, page, D, generator=g, device="cuda", dtype=torch.float32).to(dt)
        st.update(kv_len=_ints(kv), q_indptr=_ints(_indptr(q)), T=T, Q=max(q), S=max(kv), words=words,
                  scale=192 ** -0.5, pool=pool, cols=cols)
        st["mask"] = _ints(_mask_words(_parents(rng, q), q, words)) if case["tree"] else None
        st["o"] = torch.empty(T, H, kl, device="cuda", dtype=dt)
        st["lse"] = torch.empty(T, H, device="cuda")
    else:
        B, V, dt = case["B"], case["V"], DTYPES[case["dtype"]]
        q = _qlens(case)
        R, hist = sum(q), _lens(B, case["hist"])
        words, aw = -(-max(q) // 32), -(-V // 32)
        zipf = lambda *shape: (torch.rand(*shape, generator=g, device="cuda") ** 3 * V).to(torch.int32).clamp(0, V - 1)
        st["logits"] = (torch.randn(R, V, generator=g, device="cuda") * 3.0).to(dt)
        st["hist"] = zipf(B, max(hist))
        st.update(hist_len=_ints(hist), prompt_len=_ints([h // 2 for h in hist]), q_indptr=_ints(_indptr(q)))
        st["rep"] = 1.0 + 0.3 * torch.rand(B, generator=g, device="cuda")
        st["freq"] = 0.5 * torch.rand(B, generator=g, device="cuda")
        st["pres"] = 0.5 * torch.rand(B, generator=g, device="cuda")
        nb = _lens(B, case["bias"])
        st["bias_indptr"] = _ints(_indptr(nb))
        st["bias_id"] = zipf(sum(nb))
        st["bias_val"] = torch.randn(sum(nb), generator=g, device="cuda") * 2.0
        st["draft"] = zipf(R)
        st["tree"] = _ints(_mask_words(_parents(rng, q), q, words))
        # every other row is under a grammar, which allows about a third of the vocabulary
        rows = [(r // 2 if r % 2 == 0 else -1) for r in range(R)]
        st["allow_row"] = _ints(rows)
        bits = lambda: torch.randint(-2 ** 31, 2 ** 31, ((R + 1) // 2, aw), generator=g, device="cuda").to(torch.int32)
        st["allow"] = bits() & (bits() | bits())
        st.update(R=R, Q=max(q), aw=aw, words=words, out=torch.empty(R, V, device="cuda", dtype=dt))
    if own:
        _own_desc(st)
    return st


def _own_desc(st):
    """The argument blocks that a program fills once and hands over at every step."""
    import warp_b200 as wb
    wb.init(0)
    c, op = st["case"], st["case"]["op"]
    p = lambda k: st[k].data_ptr() if st[k] is not None else None
    if op == "plan":
        st["desc"] = wb.KvPlan(
            B=c["B"], T=st["T"], page=c["page"], max_blocks=st["table"].shape[1], n_free=st["free"].numel(),
            mask_words=st["words"], ctx_len=p("ctx_len"), q_len=p("q_len"), parent=p("parent"),
            free_blocks=p("free"), free_head=p("head"), n_blocks=p("held"), block_table=p("table"),
            free_head_out=p("head_out"), n_blocks_out=p("held_out"), q_indptr=p("q_indptr"),
            kv_len=p("kv_len"), pos=p("pos"), slot=p("slot"), mask=p("mask"), short_blocks=p("short"))
        st["call"] = wb.kv_plan_dev
    elif op == "rows":
        D = c["kl"] + c["rope"]
        st["desc"] = wb.MlaRows(
            T=c["T"], kl=c["kl"], rope=c["rope"], x_dtype=0, dtype=CODES[c["dtype"]], x_stride=D, x=p("x"),
            norm_w=p("w"), inv_freq=None if c["nope"] else p("inv_freq"), pos=p("pos"), slot=p("slot"),
            eps=1e-6, cache=p("cache"), row_stride=D, n_rows=st["cache"].shape[0])
        st["call"] = wb.mla_rows_dev
    elif op == "attn":
        H, D, kl = c["heads"], c["kl"] + c["rope"], c["kl"]
        ws = wb.mla_tree_ws_bytes(H, kl)
        st["ws"] = torch.empty(ws, dtype=torch.uint8, device="cuda")
        st["desc"] = wb.MlaTree(
            B=c["B"], T=st["T"], heads=H, kl=kl, rope=c["rope"], dtype=CODES[c["dtype"]], page=c["page"],
            max_blocks=st["cols"], mask_words=st["words"], n_blocks=st["pool"], row_stride=D,
            q_token_stride=H * D, q_head_stride=D, o_token_stride=H * kl, o_head_stride=kl, q=p("q"),
            cache=p("cache"), block_table=p("table"), kv_len=p("kv_len"), q_indptr=p("q_indptr"),
            mask=p("mask"), scale=st["scale"], o=p("o"), lse=p("lse"), ws=p("ws"), ws_bytes=ws)
        st["call"] = wb.mla_tree_attn_dev
    else:
        st["desc"] = wb.LogitsAdjust(
            B=c["B"], R=st["R"], V=c["V"], dtype=CODES[c["dtype"]], tree_words=st["words"],
            allow_words=st["aw"], n_allow=st["allow"].shape[0], hist_stride=st["hist"].shape[1],
            ld=c["V"], ld_out=c["V"], logits=p("logits"), out=p("out"), q_indptr=p("q_indptr"),
            hist=p("hist"), hist_len=p("hist_len"), prompt_len=p("prompt_len"), rep=p("rep"), freq=p("freq"),
            pres=p("pres"), draft=p("draft"), tree=p("tree"), bias_indptr=p("bias_indptr"),
            bias_id=p("bias_id"), bias_val=p("bias_val"), allow=p("allow"), allow_row=p("allow_row"))
        st["call"] = wb.logits_adjust_dev


# ---- one pass ------------------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if own:
        # cudaStreamLegacy (1) names the default stream; NULL would be the library's own
        st["call"](st["desc"], torch.cuda.current_stream().cuda_stream or 1)
        return _outputs(st)
    return {"plan": _plain_plan, "rows": _plain_rows, "attn": _plain_attn, "logits": _plain_logits}[op](st)


def _outputs(st):
    op = st["case"]["op"]
    if op == "plan":
        return {k: st[k] for k in ("table", "held_out", "head_out", "q_indptr", "kv_len", "pos", "slot", "mask", "short")}
    if op == "rows":
        return {"cache": st["cache"]}
    if op == "attn":
        return {"o": st["o"], "lse": st["lse"]}
    return {"out": st["out"]}


def _tokens(indptr, T):
    """The request of each of T tokens and its place there."""
    t = torch.arange(T, device="cuda")
    req = torch.searchsorted(indptr[1:].long().contiguous(), t, right=True)
    return req, t - indptr.long()[req]


def _plain_plan(st):
    c, T, Q = st["case"], st["T"], st["Q"]
    page, B = c["page"], c["B"]
    ctx, q, held = st["ctx_len"].long(), st["q_len"].long(), st["held"].long()
    need = ((ctx + q + page - 1) // page - held).clamp(min=0)
    upto = need.cumsum(0)
    avail = st["free"].numel() - st["head"].long()
    served = (upto <= avail) | (need == 0)
    given = torch.where(served, need, 0)
    first = st["head"].long() + upto - need
    col = torch.arange(st["table"].shape[1], device="cuda")[None, :] - held[:, None]
    new = (col >= 0) & (col < given[:, None])
    ids = st["free"][(first[:, None] + col).clamp(0, st["free"].numel() - 1)]
    table = torch.where(new, ids, st["table"])
    indptr = torch.cat([q.new_zeros(1), q.cumsum(0)])
    req, i = _tokens(indptr, T)
    if st["parent"] is None:
        anc = torch.tril(torch.ones(Q, Q, device="cuda")).expand(B, Q, Q)
    else:
        # the sum of a parent matrix's powers has a 1 at each ancestor: the inverse of (identity - parents)
        par = torch.zeros(B, Q, Q + 1, device="cuda")
        par[req, i, torch.where(st["parent"] < 0, Q, st["parent"]).long()] = 1.0
        eye = torch.eye(Q, device="cuda").expand(B, Q, Q)
        anc = torch.linalg.solve_triangular(eye - par[:, :, :Q], eye, upper=False)
    anc = anc[req, i].round().long()
    pos = ctx[req] + anc.sum(1) - 1
    at = ctx[req] + i
    slot = table[req, (at // page).clamp(max=table.shape[1] - 1)].long() * page + at % page
    slot = torch.where(served[req], slot, -1)
    bits = torch.nn.functional.pad(anc, (0, st["words"] * 32 - Q)).view(T, st["words"], 32)
    mask = (bits << torch.arange(32, device="cuda")).sum(2)
    mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32)
    return {"table": table, "held_out": (held + given).to(torch.int32),
            "head_out": (st["head"] + given.sum()).to(torch.int32), "q_indptr": indptr.to(torch.int32),
            "kv_len": torch.where(served, ctx + q, 0).to(torch.int32), "pos": pos.to(torch.int32), "slot": slot,
            "mask": mask, "short": (upto[-1:] - avail).clamp(min=0).to(torch.int32)}


def _plain_rows(st):
    c = st["case"]
    kl, x = c["kl"], st["x"]
    lat, r = x[:, :kl], x[:, kl:]
    lat = lat * torch.rsqrt((lat * lat).mean(1, keepdim=True) + 1e-6) * st["w"]
    if not c["nope"]:
        a = st["pos"].double()[:, None] * st["inv_freq"].double()
        cs, sn = a.cos().float(), a.sin().float()
        e, o = r[:, 0::2], r[:, 1::2]
        r = torch.stack([e * cs - o * sn, e * sn + o * cs], 2).flatten(1)
    st["cache"][st["slot"]] = torch.cat([lat, r], 1).to(st["cache"].dtype)
    return {"cache": st["cache"]}


def _plain_attn(st):
    c, T, Q, S = st["case"], st["T"], st["Q"], st["S"]
    B, H, kl, page = c["B"], c["heads"], c["kl"], c["page"]
    D = kl + c["rope"]
    ptr, kv = st["q_indptr"].long(), st["kv_len"].long()
    n = ptr[1:] - ptr[:-1]
    ctx = kv - n
    s, i = torch.arange(S, device="cuda"), torch.arange(Q, device="cuda")
    rows = st["table"].long()[:, s // page].clamp(min=0) * page + s % page
    lat = st["cache"].view(-1, D)[rows].float()                              # [B, S, D]
    qi = (ptr[:-1, None] + i).clamp(max=T - 1)
    qp = st["q"][qi].float().view(B, Q * H, D)
    j = s[None, :] - ctx[:, None]                                            # place among the new tokens
    if st["mask"] is None:
        sees = j[:, None, :] <= i[None, :, None]
    else:
        jj = j.clamp(0, st["words"] * 32 - 1)[:, None, :].expand(B, Q, S)
        word = torch.gather(st["mask"][qi].long(), 2, jj // 32)
        sees = (j[:, None, :] < 0) | ((word >> (jj % 32)) & 1).bool()
    sees = sees & (s < kv[:, None])[:, None, :]
    score = torch.matmul(qp, lat.transpose(1, 2)).view(B, Q, H, S) * st["scale"]
    score = score.masked_fill(~sees[:, :, None, :], NEG)
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == NEG, 0.0))
    total = p.sum(3, keepdim=True)
    o = torch.matmul((p / total.clamp(min=1e-38)).view(B, Q * H, S), lat[:, :, :kl]).view(B, Q, H, kl)
    lse = (top + torch.log(total))[..., 0]
    req, at = _tokens(ptr, T)
    return {"o": o[req, at].to(st["q"].dtype), "lse": lse[req, at]}


def _plain_logits(st):
    c, R, V, Q = st["case"], st["R"], st["case"]["V"], st["Q"]
    B = c["B"]
    ptr = st["q_indptr"].long()
    req, _ = _tokens(ptr, R)
    k = torch.arange(st["hist"].shape[1], device="cuda")[None, :]
    inside, said = k < st["hist_len"][:, None], k >= st["prompt_len"][:, None]
    tok = st["hist"].long()
    seen = torch.zeros(B, V, dtype=torch.int32, device="cuda").scatter_add_(1, tok, inside.int())[req]
    count = torch.zeros(B, V, dtype=torch.int32, device="cuda").scatter_add_(1, tok, (inside & said).int())[req]
    i = torch.arange(Q, device="cuda")
    node = (ptr[req][:, None] + i).clamp(max=R - 1)
    on = (((st["tree"].long()[:, i // 32] >> (i % 32)) & 1) * (i < (ptr[1:] - ptr[:-1])[req][:, None])).int()
    path = st["draft"].long()[node]
    seen.scatter_add_(1, path, on)
    count.scatter_add_(1, path, on)
    x = st["logits"].float()
    rep, freq, pres = (st[k][req][:, None] for k in ("rep", "freq", "pres"))
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * count - pres * (count > 0)
    n = st["bias_id"].numel()
    breq, _ = _tokens(st["bias_indptr"], n)
    last = torch.full((B * V,), -1, dtype=torch.int64, device="cuda")
    last.scatter_reduce_(0, breq * V + st["bias_id"].long(), torch.arange(n, device="cuda"), "amax")
    bias = torch.where(last >= 0, st["bias_val"][last.clamp(min=0)], 0.0).view(B, V)
    x = x + bias[req]
    bits = (st["allow"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    bits = bits.view(st["allow"].shape[0], -1)[:, :V].bool()
    rows = st["allow_row"].long()
    ok = bits[rows.clamp(min=0)] | (rows < 0)[:, None]
    return {"out": torch.where(ok, x, NEG).to(st["logits"].dtype)}


# ---- what a pass cannot do without ---------------------------------------------------------------------

def work(case):
    op, size = case["op"], {"f32": 4, "f16": 2, "bf16": 2}
    if op == "plan":
        q, B, page = _qlens(case), case["B"], case["page"]
        T, words = sum(q), -(-max(q) // 32)
        new = sum(max(0, _padded(c + n, page) - _padded(c, page)) for c, n in zip(_lens(B, case["ctx"]), q))
        # lengths and counts in and out, the taken blocks' ids in and out, a table entry in and a position, a
        # slot and a mask out for each token
        return {"bytes": 24 * B + 8 * new + T * (4 + 4 + 8 + 4 * words + (4 if case["tree"] else 0)), "flops": 8 * T}
    if op == "rows":
        T, D = case["T"], case["kl"] + case["rope"]
        return {"bytes": T * (D * (4 + size[case["dtype"]]) + 12), "flops": T * (4 * case["kl"] + 6 * case["rope"])}
    q = _qlens(case)
    if op == "attn":
        H, kl, D, z = case["heads"], case["kl"], case["kl"] + case["rope"], size[case["dtype"]]
        kv = [c + n for c, n in zip(_lens(case["B"], case["ctx"]), q)]
        # a chain's token sees the cached rows and those up to its own; a tree's at most as many
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(q, kv))
        return {"bytes": z * (sum(kv) * D + sum(q) * H * (D + kl)) + 4 * sum(q) * H,
                "flops": 2 * pairs * H * (D + kl)}
    R, V, z = sum(q), case["V"], size[case["dtype"]]
    return {"bytes": 2 * R * V * z + (R + 1) // 2 * V // 8 + 4 * sum(_lens(case["B"], case["hist"])),
            "flops": 6 * R * V}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    st = prepare(case, seed)
    own = was
    op = case["op"]
    if op == "plan":
        return None                              # whole numbers only
    if op == "rows":
        kl = case["kl"]
        out = st["cache"].double()
        x = st["x"].double()
        lat = x[:, :kl]
        rms = ((lat ** 2).sum(1) / kl + float(torch.tensor(1e-6))).sqrt()
        rot = torch.view_as_complex(x[:, kl:].reshape(case["T"], -1, 2).contiguous())
        if not case["nope"]:
            angle = torch.outer(st["pos"].double(), st["inv_freq"].double())
            rot = rot * torch.polar(torch.ones_like(angle), angle)
        out[st["slot"]] = torch.cat([lat / rms[:, None] * st["w"].double(), torch.view_as_real(rot).flatten(1)], 1)
        return {"cache": out}
    ptr = st["q_indptr"].tolist()
    if op == "attn":
        H, kl, page = case["heads"], case["kl"], case["page"]
        if work(case)["flops"] > 3e12:
            return None
        o = torch.zeros(st["T"], H, kl, dtype=torch.float64, device="cuda")
        lse = torch.full((st["T"], H), NEG, dtype=torch.float64, device="cuda")
        for r, n in enumerate(st["kv_len"].tolist()):
            a, b = ptr[r], ptr[r + 1]
            c = n - (b - a)
            lat = st["cache"][st["table"][r, :_padded(n, page)].long()].flatten(0, 1)[:n].double()
            for t0 in range(a, b, 16):
                t1 = min(b, t0 + 16)
                if st["mask"] is None:
                    see = torch.arange(n, device="cuda")[None, :] <= c + torch.arange(t0 - a, t1 - a, device="cuda")[:, None]
                else:
                    see = torch.ones(t1 - t0, n, dtype=torch.bool, device="cuda")
                    words = [[w & 0xFFFFFFFF for w in row] for row in st["mask"][t0:t1].tolist()]
                    see[:, c:] = torch.tensor([[bool(row[k // 32] >> (k % 32) & 1) for k in range(b - a)] for row in words],
                                              device="cuda")
                s = torch.einsum("thd,sd->ths", st["q"][t0:t1].double(), lat) * st["scale"]
                s = torch.where(see[:, None, :], s, NEG)
                z = torch.logsumexp(s, 2)
                o[t0:t1] = torch.einsum("ths,sd->thd", torch.exp(s - z[:, :, None]), lat[:, :kl])
                lse[t0:t1] = z
        return {"o": o, "lse": lse}
    V = case["V"]
    out = st["logits"].double()
    blist = st["bias_indptr"].tolist()
    for r in range(case["B"]):
        n, m = int(st["hist_len"][r]), int(st["prompt_len"][r])
        everything = torch.bincount(st["hist"][r, :n].long(), minlength=V)
        said = torch.bincount(st["hist"][r, m:n].long(), minlength=V)
        bias = dict(zip(st["bias_id"][blist[r]:blist[r + 1]].tolist(), st["bias_val"][blist[r]:blist[r + 1]].tolist()))
        for t in range(ptr[r], ptr[r + 1]):
            row = [w & 0xFFFFFFFF for w in st["tree"][t].tolist()]
            nodes = [k for k in range(ptr[r + 1] - ptr[r]) if row[k // 32] >> (k % 32) & 1]
            mine = torch.bincount(st["draft"][ptr[r]:ptr[r + 1]].long()[nodes], minlength=V)
            x, rep = out[t], st["rep"][r].double()
            x = torch.where(everything + mine > 0, torch.where(x > 0, x / rep, x * rep), x)
            x = x - st["freq"][r].double() * (said + mine) - st["pres"][r].double() * (said + mine > 0)
            x[torch.tensor(list(bias), device="cuda")] += torch.tensor(list(bias.values()), dtype=torch.float64, device="cuda")
            a = int(st["allow_row"][t])
            if a >= 0:
                v = torch.arange(V, device="cuda")
                x = torch.where((st["allow"][a].long()[v // 32] >> (v % 32)) & 1 == 1, x, NEG)
            out[t] = x
    return {"out": out}
