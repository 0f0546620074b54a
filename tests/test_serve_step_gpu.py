"""The serving step's operators on the device (warp_b200/csrc/serve_step.cu,
mla_tree.cu) against their 64-bit definitions in serve_oracle.py, at the
sizes, masks and layouts where they can go wrong, and run together.

Tolerances are the ones derived beside the oracle, before any run: whole
numbers are equal, rounded values within half a step of their type plus the
bound on the 32-bit sums behind them."""
import random

import numpy as np
import pytest
import torch

import serve_oracle as O
from serve_oracle import CODE, DT, HALF, TINY

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).cuda()


def u32(x):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.uint32)).view(np.int32)).cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def p(t):
    return t.data_ptr() if t is not None else None


def parents(rng, q):
    out = []
    for n in q:
        out += [-1 if i == 0 or rng.random() < 0.1 else rng.randrange(i) for i in range(n)]
    return out


def ancestors(par, q, words):
    rows, at = [], 0
    for n in q:
        bits = []
        for i in range(n):
            a = par[at + i]
            bits.append((bits[a] if a >= 0 else 0) | 1 << i)
        rows += [[(b >> 32 * w) & 0xFFFFFFFF for w in range(words)] for b in bits]
        at += n
    return np.array(rows, np.uint32).reshape(-1, words)


# ---- plan ----------------------------------------------------------------------------

class Plan:
    def __init__(self, wb, ctx, q, held, table, free, head, page, words, parent, extra=3, masked=True, inplace=False):
        B, T = len(ctx), sum(q)
        self.T = T + extra
        self.t = dict(ctx_len=dev(ctx), q_len=dev(q), parent=dev(parent) if parent is not None else None,
                      free_blocks=dev(free if len(free) else [0]), free_head=dev([head]), n_blocks=dev(held),
                      block_table=dev(table), q_indptr=dev([-7] * (B + 1)), kv_len=dev([-7] * B),
                      pos=dev([-7] * self.T), slot=dev([-7] * self.T, torch.int64),
                      mask=dev(np.full((self.T, words), -7)) if masked else None, short_blocks=dev([-7]))
        self.t["free_head_out"] = self.t["free_head"] if inplace else dev([-7])
        self.t["n_blocks_out"] = self.t["n_blocks"] if inplace else dev([-7] * B)
        self.d = wb.KvPlan(B=B, T=self.T, page=page, max_blocks=np.asarray(table).shape[1], n_free=len(free),
                           mask_words=words, **{k: p(v) for k, v in self.t.items()})

    def check(self, ref):
        g = {k: v.cpu().numpy() if v is not None else None for k, v in self.t.items()}
        n = len(ref["pos"])
        assert g["q_indptr"].tolist() == ref["q_indptr"]
        assert g["kv_len"].tolist() == ref["kv_len"]
        assert g["n_blocks_out"].tolist() == ref["n_blocks"]
        assert g["free_head_out"].tolist() == [ref["head"]]
        assert g["short_blocks"].tolist() == [ref["short"]]
        assert np.array_equal(g["block_table"], ref["table"])
        assert g["pos"].tolist() == ref["pos"] + [-7] * (self.T - n)
        assert g["slot"].tolist() == ref["slot"] + [-7] * (self.T - n)
        if g["mask"] is not None:
            assert np.array_equal(g["mask"][:n].view(np.uint32), ref["mask"])
            assert (g["mask"][n:] == -7).all()


def plan_case(seed, B, ctx_most, q_most, page, tree, short):
    rng = random.Random(seed)
    ctx = [rng.choice([0, 1, page - 1, page, page + 1, rng.randrange(ctx_most + 1)]) for _ in range(B)]
    q = [rng.choice([0, 1, 1, rng.randrange(q_most + 1), q_most]) for _ in range(B)]
    held = [-(-c // page) + rng.choice([0, 0, 1]) for c in ctx]
    cols = max(max(-(-(c + n) // page) for c, n in zip(ctx, q)), max(held)) + 2
    need = sum(max(0, -(-(c + n) // page) - h) for c, n, h in zip(ctx, q, held))
    ids = list(range(sum(held) + need + 5))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-9] * (cols - h))
        at += h
    head = 2
    free = [-1, -1] + ids[at:at + max(0, need + (3 if not short else -short))]
    words = -(-max(1, q_most) // 32)
    return ctx, q, held, table, free, head, page, words, parents(rng, q) if tree else None


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("seed,B,ctx,q,page,tree,short", [
    (1, 1, 0, 1, 1, False, 0), (2, 1, 100, 1, 16, True, 0), (3, 5, 40, 7, 4, True, 0), (4, 33, 300, 33, 16, True, 2),
    (5, 64, 4096, 1, 64, False, 0), (6, 600, 900, 9, 32, True, 5), (7, 17, 50, 70, 24, False, 0),
    (8, 4096, 64, 3, 8, True, 1), (9, 3, 5000, 4000, 16, False, 0), (10, 9, 64, 64, 16, True, 10 ** 6)])
def test_plan(cuda_lib, seed, B, ctx, q, page, tree, short, inplace):
    c = plan_case(seed, B, ctx, q, page, tree, short)
    pl = Plan(cuda_lib, *c, inplace=inplace)
    cuda_lib.kv_plan_dev(pl.d, stream())
    torch.cuda.synchronize()
    pl.check(O.plan(c[0], c[1], c[2], c[3], c[4], c[5], c[6], pl.T, c[7], c[8], len(c[3][0])))
    assert cuda_lib.device_errors() == 0


def test_plan_steps(cuda_lib):
    """Steps in place on one set of arrays, captured once and replayed with new
    lengths: the blocks each request holds follow the definition's."""
    rng = random.Random(3)
    B, page, cols = 12, 8, 20
    held, table, free, head = [0] * B, np.full((B, cols), -1), list(range(300)), 0
    rng.shuffle(free)
    ctx = [0] * B
    q = [5] * B
    pl = Plan(cuda_lib, ctx, q, held, table, free, head, page, 1, None, extra=0, inplace=True)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cuda_lib.kv_plan_dev(pl.d, stream())
    for step in range(9):
        ref = O.plan(ctx, q, held, table, free, head, page, pl.T, 1, None, cols)
        pl.t["ctx_len"].copy_(dev(ctx))
        pl.t["q_len"].copy_(dev(q))
        for k in ("pos", "slot", "mask"):
            pl.t[k].fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        pl.check(ref)
        held, table, head = ref["n_blocks"], ref["table"], ref["head"]
        # some of the new tokens are kept, as after drafts were checked
        ctx = [c + rng.randrange(n + 1) for c, n in zip(ctx, q)]
        q = [rng.randrange(6) for _ in range(B)]


def test_plan_without_mask(cuda_lib):
    c = plan_case(11, 7, 90, 100, 16, False, 0)
    pl = Plan(cuda_lib, *c, masked=False)
    cuda_lib.kv_plan_dev(pl.d, stream())
    torch.cuda.synchronize()
    pl.check(O.plan(c[0], c[1], c[2], c[3], c[4], c[5], c[6], pl.T, c[7], None, len(c[3][0]), masked=False))
    assert cuda_lib.device_errors() == 0


def test_plan_reports(cuda_lib):
    """Trees and lengths out of range: reported, the request left out, the
    others served."""
    wb = cuda_lib
    table = np.full((3, 4), -1)
    pl = Plan(wb, [0, 4, 8], [2, 40, 1], [0, 1, 2], table, list(range(50)), 0, 4, 1, [-1] * 43, extra=0)
    wb.kv_plan_dev(pl.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_BLOCK | wb.DERR_BAD_TREE        # 40 nodes: 11 blocks, 2 words
    assert pl.t["kv_len"].tolist() == [2, 0, 9] and pl.t["n_blocks_out"].tolist() == [1, 1, 3]
    assert pl.t["slot"].tolist()[2:42] == [-1] * 40 and pl.t["slot"].tolist()[42] == 1 * 4 + 0
    pl = Plan(wb, [0, -5], [3, 1], [0, 0], np.full((2, 4), -1), [3, 1], 0, 4, 1, [-1, 2, 0, -1], extra=0)
    wb.kv_plan_dev(pl.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_BLOCK | wb.DERR_BAD_TREE        # a parent that is no earlier node
    assert pl.t["kv_len"].tolist() == [3, 0] and pl.t["pos"].tolist()[:3] == [0, 0, 1]
    # more tokens than rows: the rows there are get theirs
    pl = Plan(wb, [0, 0], [3, 3], [0, 0], np.full((2, 2), -1), [5, 6], 0, 4, 1, None, extra=-2)
    wb.kv_plan_dev(pl.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_TREE
    assert pl.t["q_indptr"].tolist() == [0, 3, 4] and pl.t["slot"].tolist() == [20, 21, 22, 24]


def test_plan_tree_too_large(cuda_lib):
    """A chain of nodes far past the mask's words: reported and not served, and
    the nodes without a bit are not walked up from (their pos is the request's
    length)."""
    wb = cuda_lib
    pl = Plan(wb, [5], [100], [2], np.full((1, 40), -1), list(range(50)), 0, 4, 1, [i - 1 for i in range(100)], extra=0)
    wb.kv_plan_dev(pl.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_TREE
    assert pl.t["kv_len"].tolist() == [0] and pl.t["slot"].tolist() == [-1] * 100
    assert pl.t["pos"].tolist() == [5 + i for i in range(32)] + [5] * 68


@pytest.mark.parametrize("head,taken", [(-1, [4]), (5, [-1]), (2 ** 31 - 1, [-1]), (-2 ** 31, [4])])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan_free_head_outside(cuda_lib, head, taken, inplace):
    """A head outside the free list is reported; requests that hold their
    blocks are served all the same."""
    wb = cuda_lib
    pl = Plan(wb, [3, 2, 1], [1, 3, 1], [1, 1, 1], [[9, -1], [8, -1], [3, -1]], [4, 5, 6, 7], head, 4, 1, None, extra=0, inplace=inplace)
    wb.kv_plan_dev(pl.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_BLOCK
    assert pl.t["kv_len"].tolist() == [4, 5 if taken[0] >= 0 else 0, 2]
    assert pl.t["block_table"].tolist() == [[9, -1], [8] + taken, [3, -1]]
    assert pl.t["free_head_out"].tolist() == [1 if head < 0 else head]
    assert pl.t["short_blocks"].tolist() == [0 if head < 0 else 1]


# ---- rows ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("xdtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,kl,rope,pad,nope", [
    (1, 512, 64, 0, False), (7, 512, 64, 5, True), (130, 64, 16, 0, False), (33, 500, 62, 3, False),
    (5, 4096, 512, 0, False), (3, 1, 0, 0, True), (6, 512, 0, 1, False)])
def test_rows(cuda_lib, T, kl, rope, pad, nope, dtype, xdtype):
    g = torch.Generator().manual_seed(T * 1000 + kl)
    D, n = kl + rope, T + 9
    x = torch.randn(T, D + pad, generator=g).to(DT[xdtype])
    w = 1 + 0.3 * torch.randn(kl, generator=g)
    inv = None if nope else 10000.0 ** (-torch.arange(0, rope, 2).float() / max(rope, 1))
    pos = torch.randint(0, 1 << 21, (T,), generator=g, dtype=torch.int32)
    slot = torch.randperm(n, generator=g)[:T]
    if T > 2:
        slot[1] = -1                               # a token that was not served
    cache = torch.randn(n, D + pad, generator=g).to(DT[dtype])
    c, xs, ws, ps, ss = cache.cuda(), x.cuda(), w.cuda(), pos.cuda(), slot.cuda()
    iv = inv.cuda() if inv is not None else None
    cuda_lib.mla_rows_dev(cuda_lib.MlaRows(
        T=T, kl=kl, rope=rope, x_dtype=CODE[xdtype], dtype=CODE[dtype], x_stride=D + pad, x=p(xs), norm_w=p(ws),
        inv_freq=p(iv) if rope else None, pos=p(ps), slot=p(ss), eps=1e-6, cache=p(c), row_stride=D + pad, n_rows=n), stream())
    got = c.cpu()
    ref = O.rows(x[:, :D], w, inv if rope else None, pos, 1e-6)
    keep = torch.ones(n, dtype=torch.bool)
    keep[slot[slot >= 0]] = False
    assert torch.equal(got[keep], cache[keep])                     # other rows as they were
    assert torch.equal(got[:, D:], cache[:, D:])                   # and what lies between rows
    # the sum of kl squares is off by kl e of itself, its root by half of that; five more roundings.
    # rotated: the float angle in [-pi, pi] is off by pi e (2 e pi with the turn's), sin and cos by 2 e
    for t in range(T):
        if slot[t] < 0:
            continue
        d = (got[slot[t], :D].double() - ref[t]).abs()
        tol = ref[t].abs() * (HALF[dtype] + (kl / 2 + 8) * E) + TINY[dtype]
        size = x[t, kl:D].double().abs().view(-1, 2).sum(1).repeat_interleave(2) if rope else x.new_zeros(0).double()
        tol[kl:] += 12 * E * size
        assert bool((d <= tol).all()), float((d / tol).max())
    assert cuda_lib.device_errors() == 0


def test_rows_slot_outside(cuda_lib):
    wb = cuda_lib
    x, w = torch.randn(2, 80).cuda(), torch.ones(64).cuda()
    c = torch.zeros(4, 80).cuda()
    slot = dev([4, 1], torch.int64)
    wb.mla_rows_dev(wb.MlaRows(T=2, kl=64, rope=16, x_dtype=0, dtype=0, x_stride=80, x=p(x), norm_w=p(w), slot=p(slot),
                               eps=1e-6, cache=p(c), row_stride=80, n_rows=4), stream())
    assert wb.device_errors() == wb.DERR_BAD_BLOCK
    assert bool((c[[0, 2, 3]] == 0).all()) and bool((c[1] != 0).any())


# ---- attention -----------------------------------------------------------------------

class Attn:
    """One call's arrays. ctx, q: lengths; unserved: requests whose kv_len is 0."""

    def __init__(self, wb, seed, dtype, H, kl, rope, page, ctx, q, tree=None, pad=0, unserved=(), spare=3, extra=2,
                 lse=True, blocks_at=0):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.args = dict(kl=kl, page=page, dtype=dtype)
        self.H, self.D, self.kl, self.rope, self.dtype, self.wb = H, kl + rope, kl, rope, dtype, wb
        self.kv = [0 if r in unserved else c + n for r, (c, n) in enumerate(zip(ctx, q))]
        self.indptr = [0]
        for n in q:
            self.indptr.append(self.indptr[-1] + n)
        self.T = self.indptr[-1]
        need = [-(-k // page) for k in self.kv]
        cols = max(1, max(need))
        ids = list(range(blocks_at, blocks_at + sum(need) + spare))
        rng.shuffle(ids)
        self.table, at = np.full((len(q), cols), -1, np.int64), 0
        for r, n in enumerate(need):
            self.table[r, :n] = ids[at:at + n]
            at += n
        self.n_blocks = blocks_at + sum(need) + spare
        D, dt = self.D, DT[dtype]
        self.q = (torch.randn(self.T + extra, H, D + pad, generator=g) * 1.5).to(dt)
        self.cache = torch.randn(self.n_blocks - blocks_at, page, D + pad, generator=g).to(dt)
        words = -(-max(1, max(q)) // 32)
        self.mask = None
        if tree is not None:
            self.mask = tree if isinstance(tree, np.ndarray) else ancestors(parents(rng, q), q, words)
        self.scale, self.page, self.words, self.blocks_at, self.pad = 0.11, page, words, blocks_at, pad
        self.extra, self.want_lse = extra, lse

    def put(self):
        wb, H, D, kl, pad = self.wb, self.H, self.D, self.kl, self.pad
        self.gc = self.cache.cuda()
        self.gq = self.q.cuda()
        self.go = torch.full((self.T + self.extra, H, kl + pad), 7.0, dtype=DT[self.dtype], device="cuda")
        self.gl = torch.full((self.T + self.extra, H), 7.0, device="cuda") if self.want_lse else None
        self.gm = u32(self.mask) if self.mask is not None else None
        self.gt, self.gk, self.gi = dev(self.table), dev(self.kv), dev(self.indptr)
        n = wb.mla_tree_ws_bytes(H, kl)
        # whatever an earlier call left there
        self.ws = torch.full((n // 4,), float("nan"), device="cuda")
        cache = p(self.gc) - self.blocks_at * self.page * (D + pad) * self.gc.element_size()
        self.d = wb.MlaTree(B=len(self.kv), T=self.T + self.extra, heads=H, kl=kl, rope=self.rope, dtype=CODE[self.dtype],
                            page=self.page, max_blocks=self.table.shape[1], mask_words=self.words, n_blocks=self.n_blocks,
                            row_stride=D + pad, q_token_stride=H * (D + pad), q_head_stride=D + pad,
                            o_token_stride=H * (kl + pad), o_head_stride=kl + pad, q=p(self.gq), cache=cache,
                            block_table=p(self.gt), kv_len=p(self.gk), q_indptr=p(self.gi), mask=p(self.gm),
                            scale=self.scale, o=p(self.go), lse=p(self.gl), ws=p(self.ws), ws_bytes=n)
        return self

    def call(self):
        self.wb.mla_tree_attn_dev(self.d, stream())
        return self

    def ref(self):
        c = self.cache[:, :, :self.D]
        return O.attn(self.q[:self.T, :, :self.D], c, self.table - self.blocks_at, self.kv, self.indptr, self.mask,
                      self.scale, self.kl, self.page, self.dtype)

    def check(self, ref=None):
        torch.cuda.synchronize()
        o, lse, to, tl = ref or self.ref()
        got = self.go.cpu()
        if self.T:
            d = (got[:self.T, :, :self.kl].double() - o).abs()
            assert bool((d <= to).all()), ("o", float((d / to.clamp(min=1e-30)).max()), int((~(d <= to)).sum()))
        assert bool((got[self.T:] == 7).all()) and bool((got[:, :, self.kl:] == 7).all())
        if self.gl is not None:
            l = self.gl.cpu().double()
            assert bool((l[self.T:] == 7).all())
            l = l[:self.T]
            assert torch.equal(torch.isinf(l), torch.isinf(lse))
            fin = ~torch.isinf(lse)
            assert bool(((l - lse).abs()[fin] <= tl[fin]).all())
        assert self.wb.device_errors() == 0
        return self


KIMI = (512, 64)
ATTN = {
    # name: (dtype, heads, (kl, rope), page, ctx, q, tree)
    "one_row": ("bf16", 32, KIMI, 64, [0], [1], None),
    "one_head": ("bf16", 1, KIMI, 16, [5], [1], None),
    "tile_edges": ("bf16", 32, KIMI, 64, [126, 127, 128, 255, 63, 64], [1] * 6, None),
    "ragged": ("bf16", 32, KIMI, 64, [0, 1, 700, 0, 333], [1, 0, 1, 3, 2], None),
    "tree": ("bf16", 32, KIMI, 16, [300, 0, 128, 1], [7, 5, 16, 1], 1),
    "tree_wide": ("f16", 32, KIMI, 32, [90], [64], 1),
    "tree_wider": ("bf16", 4, KIMI, 64, [130, 2], [70, 33], 1),
    "chain": ("f16", 32, KIMI, 64, [0, 40], [70, 9], None),
    "prompt": ("bf16", 16, KIMI, 128, [0], [300], None),
    "heads_20": ("bf16", 20, KIMI, 32, [200, 77], [3, 5], 1),
    "heads_64": ("f16", 64, KIMI, 64, [150], [3], None),
    "heads_128": ("bf16", 128, KIMI, 64, [200], [1], None),
    "long": ("bf16", 32, KIMI, 64, [6000], [2], None),
    "long_few": ("f16", 8, KIMI, 8, [5000, 3], [1, 1], None),
    "pages_24": ("bf16", 32, KIMI, 24, [200, 31], [4, 1], 1),
    "pages_8": ("f16", 32, KIMI, 8, [133], [2], None),
    "pages_256": ("bf16", 32, KIMI, 256, [300, 255], [2, 1], None),
    "pages_1": ("bf16", 32, KIMI, 1, [130], [2], None),
    "pages_5": ("f16", 4, KIMI, 5, [77, 4], [3, 1], 1),
    "kl_128": ("bf16", 16, (128, 16), 16, [260, 9], [5, 1], 1),
    "kl_256": ("f16", 32, (256, 32), 32, [130], [4], None),
    "kl_384_no_rope": ("bf16", 32, (384, 0), 64, [200], [2], None),
    "kl_64": ("bf16", 4, (64, 16), 16, [140], [3], 1),
    "kl_odd": ("f16", 3, (77, 5), 16, [90], [3], None),
    "kl_1": ("f32", 2, (1, 0), 4, [9], [2], None),
    "rope_128": ("bf16", 8, (512, 128), 64, [150], [2], None),
    # several key tiles a CTA, tiles cut between CTAs, of one, two and three tokens' rows
    "many_singles": ("bf16", 32, KIMI, 64, [900 - 37 * r for r in range(24)] * 2, [1] * 48, None),
    "many_pairs": ("f16", 32, KIMI, 32, [1500 - 90 * r for r in range(16)] * 2, [2] * 32, 1),
    "many_drafts": ("bf16", 32, KIMI, 64, [2900 - 200 * r for r in range(12)], [5, 3, 4, 9] * 3, 1),
    "many_chunks": ("f16", 32, KIMI, 16, [1500, 0, 900, 1200], [40, 100, 33, 20], None),
    "many_narrow": ("bf16", 64, (192, 32), 64, [2600 - 170 * r for r in range(12)], [3, 2] * 6, 1),
    "many_small_pages": ("bf16", 32, KIMI, 4, [1300 - 100 * r for r in range(12)], [3, 1, 2, 4] * 3, 1),
    "many_f32": ("f32", 16, (128, 16), 16, [1700 - 100 * r for r in range(16)], [1, 2] * 8, 1),
    "f32_engine": ("f32", 32, KIMI, 64, [500], [1], None),
    "f32_tree": ("f32", 32, KIMI, 16, [90, 0, 200], [5, 3, 1], 1),
    "f32_small": ("f32", 4, (64, 16), 16, [33, 64, 0], [2, 1, 4], None),
}


def attn_case(wb, name, seed=None, **kw):
    dtype, H, (kl, rope), page, ctx, q, tree = ATTN[name]
    return Attn(wb, seed or len(name) * 37 + sum(ctx), dtype, H, kl, rope, page, ctx, q, tree, **kw)


@pytest.mark.parametrize("name", list(ATTN))
def test_attn(cuda_lib, name):
    attn_case(cuda_lib, name).put().call().check()


@pytest.mark.parametrize("name", ["tree", "ragged", "f32_tree", "kl_64", "kl_128"])
@pytest.mark.parametrize("pad", [8, 3])
def test_attn_strides(cuda_lib, name, pad):
    """Rows, heads and outputs apart; 8 keeps 16-byte rows, 3 leaves none."""
    attn_case(cuda_lib, name, pad=pad).put().call().check()


@pytest.mark.parametrize("name", ["tree", "f32_tree", "chain"])
def test_attn_head_major(cuda_lib, name):
    """q and o as [heads][tokens][...]: the token stride below the head stride."""
    a = attn_case(cuda_lib, name, extra=0).put()
    a.gq = a.gq.transpose(0, 1).contiguous()
    out = torch.zeros(a.H, a.T, a.kl, dtype=DT[a.dtype], device="cuda")
    a.d.q, a.d.q_token_stride, a.d.q_head_stride = p(a.gq), a.D, a.T * a.D
    a.d.o, a.d.o_token_stride, a.d.o_head_stride = p(out), a.kl, a.T * a.kl
    a.call()
    a.go = out.transpose(0, 1)
    a.check()


@pytest.mark.parametrize("name", ["tree", "f32_tree", "long"])
def test_attn_unserved_and_empty(cuda_lib, name):
    """A request that was not served, tokens whose mask is empty (one of them
    with nothing cached either), no lse."""
    dtype, H, (kl, rope), page, ctx, q, tree = ATTN[name]
    ctx, q = [0] + ctx + [40], [2] + q + [3]
    mask = ancestors([i - 1 for n in q for i in range(n)], q, -(-max(q) // 32))
    mask[0] = 0
    mask[3] = 0
    a = Attn(cuda_lib, 5, dtype, H, kl, rope, page, ctx, q, mask, unserved=(len(q) - 1,)).put().call().check()
    assert bool((a.go[0] == 0).all()) and bool(torch.isinf(a.gl[0]).all())
    assert bool((a.go[a.T - 3:a.T] == 0).all())
    b = Attn(cuda_lib, 5, dtype, H, kl, rope, page, ctx, q, mask, unserved=(len(q) - 1,), lse=False).put().call()
    torch.cuda.synchronize()
    assert torch.equal(a.go, b.go)


@pytest.mark.parametrize("name", ["tree", "f32_tree", "pages_24", "pages_5", "kl_128", "tile_edges", "many_singles",
                                  "many_pairs", "many_drafts", "many_small_pages", "many_f32"])
def test_attn_what_is_not_seen(cuda_lib, name):
    """NaN and infinities in rows behind a request's last, in blocks of no
    request, behind the latents of a row, and in a drafted row that only some
    tokens see, reach only who sees them."""
    a = attn_case(cuda_lib, name, pad=8)
    ref = a.ref()
    used = np.zeros((a.n_blocks, a.page), bool)
    for r, n in enumerate(a.kv):
        for k in range(n):
            used[a.table[r, k // a.page], k % a.page] = True
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")])
    a.cache[torch.from_numpy(~used)] = bad[torch.arange(int((~used).sum())) % 3][:, None].to(a.cache.dtype)
    a.cache[:, :, a.D:] = float("nan")
    a.put().call().check(ref)
    if a.mask is None:
        return
    # a drafted row of NaN in each request that drafts several tokens
    spoiled = torch.zeros(a.T, dtype=torch.bool)
    for r in range(len(a.kv)):
        n = a.indptr[r + 1] - a.indptr[r]
        if n < 2:
            continue
        j = n - 2
        k = a.kv[r] - n + j
        a.cache[a.table[r, k // a.page], k % a.page, (r * 7) % a.D] = [float("nan"), float("inf")][r % 2]
        for t in range(a.indptr[r], a.indptr[r + 1]):
            spoiled[t] = bool((int(a.mask[t][j // 32]) >> (j % 32)) & 1)
    assert bool(spoiled.any()) and not bool(spoiled.all())
    a.put().call()
    torch.cuda.synchronize()
    o, _, to, _ = ref
    clean = ~spoiled
    d = (a.go[:a.T, :, :a.kl].cpu().double() - o).abs()[clean]
    assert bool((d <= to[clean]).all())


@pytest.mark.parametrize("name", ["tree", "long", "f32_tree", "many_singles", "many_pairs", "many_drafts", "many_f32"])
def test_attn_extreme_scores(cuda_lib, name):
    """Scores of some thousands, of both signs, rising along the cache: the
    softmax stays finite and is the largest key's."""
    a = attn_case(cuda_lib, name)
    ramp = torch.linspace(0.25, 8.0, a.cache.shape[0] * a.page).view(-1, a.page, 1)
    a.cache = (a.cache.float() * ramp).to(a.cache.dtype)
    a.q = (a.q.float() * 16).to(a.q.dtype)
    a.put().call().check()
    a.d.scale = a.scale = -a.scale
    a.call().check()


@pytest.mark.parametrize("name", ["tree", "many_singles", "f32_tree"])
def test_attn_scale_zero(cuda_lib, name):
    """All seen rows weigh the same; masked ones nothing."""
    a = attn_case(cuda_lib, name)
    a.scale = 0.0
    a.put().call().check()


def test_attn_two_threads(cuda_lib):
    """Calls from two host threads, each on its stream with its workspace."""
    import threading
    cases = [attn_case(cuda_lib, "many_pairs").put(), attn_case(cuda_lib, "many_singles").put()]
    refs = [c.ref() for c in cases]

    def run(c):
        torch.cuda.set_device(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                c.call()
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    ts = [threading.Thread(target=run, args=(c,)) for c in cases]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    for c, ref in zip(cases, refs):
        c.check(ref)


def test_attn_nan_query(cuda_lib):
    """A NaN in one query row stays in its row."""
    for name in ("tree", "f32_tree"):
        a = attn_case(cuda_lib, name)
        ref = a.ref()
        a.q[1, 1, 3] = float("nan")
        a.put().call()
        torch.cuda.synchronize()
        got = a.go[:a.T, :, :a.kl].cpu().double()
        assert bool(torch.isnan(got[1, 1]).all())
        got[1, 1] = ref[0][1, 1]
        assert bool(((got - ref[0]).abs() <= ref[2]).all())


@pytest.mark.parametrize("dtype,page", [("bf16", 64), ("f32", 64), ("f16", 5)])
def test_attn_far_blocks(cuda_lib, dtype, page):
    """Blocks whose element offsets pass 2^32 (the cache's address is set so
    that only the far end of it exists)."""
    far = (1 << 32) // (page * 576) + 11
    a = Attn(cuda_lib, 9, dtype, 32, 512, 64, page, [150, 70], [2, 1], None, blocks_at=0)
    a.blocks_at = 0
    z = 2 if dtype != "f32" else 4
    big = torch.empty(((far + a.n_blocks) * page * 576 * z,), dtype=torch.uint8, device="cuda")
    a.put()
    view = big.view(DT[dtype]).view(-1, page, 576)
    view[far:far + a.n_blocks] = a.gc
    a.gt += torch.where(a.gt >= 0, far, 0).to(torch.int32)
    a.d.cache, a.d.n_blocks = p(big), far + a.n_blocks
    a.call().check()


@pytest.mark.parametrize("name", ["tree", "f32_tree"])
def test_attn_bad_blocks(cuda_lib, name):
    """A block id outside the cache and a length beyond the table are
    reported; nothing outside is touched."""
    wb = cuda_lib
    a = attn_case(wb, name).put()
    ref = a.ref()
    for bad in (a.n_blocks, -3, 2 ** 31 - 1):
        a.gt = dev(a.table)
        a.gt[0, 1] = bad
        a.d.block_table = p(a.gt)
        a.call()
        torch.cuda.synchronize()
        assert wb.device_errors() == wb.DERR_BAD_BLOCK
        rest = slice(a.indptr[1], a.T)
        assert bool(((a.go[rest, :, :a.kl].cpu().double() - ref[0][rest]).abs() <= ref[2][rest]).all())
    a.gt = dev(a.table)
    a.d.block_table = p(a.gt)
    a.gk[0] = a.table.shape[1] * a.page + 1
    a.call()
    assert wb.device_errors() == wb.DERR_BAD_BLOCK


@pytest.mark.parametrize("name", ["long", "tree", "f32_tree", "prompt", "many_singles", "many_pairs", "many_drafts",
                                  "many_chunks", "many_f32"])
def test_attn_same_every_time(cuda_lib, name):
    """The same bits from every call, and beside calls on another stream."""
    a, b = attn_case(cuda_lib, name).put(), attn_case(cuda_lib, "ragged").put()
    a.call()
    torch.cuda.synchronize()
    first, fl = a.go.clone(), a.gl.clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        a.go.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            a.call()
        with torch.cuda.stream(s2):
            b.call()
        torch.cuda.synchronize()
        assert torch.equal(a.go, first) and torch.equal(a.gl, fl)


def test_attn_graphs(cuda_lib):
    """Two captured calls, each with its own workspace, replayed at once with
    new lengths and tables."""
    a, b = attn_case(cuda_lib, "long").put(), attn_case(cuda_lib, "tree").put()
    graphs = []
    for c in (a, b):
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=s):
            c.call()
        graphs.append((g, s))
    for shorter in (0, 1, 2):
        for c in (a, b):
            c.kv = [k - shorter if k - shorter >= c.indptr[r + 1] - c.indptr[r] else k for r, k in enumerate(c.kv)]
            c.gk.copy_(dev(c.kv))
            c.go.fill_(7.0)
        torch.cuda.synchronize()
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        a.check()
        b.check()


def test_attn_workspace_too_small(cuda_lib):
    a = attn_case(cuda_lib, "tree").put()
    a.d.ws_bytes -= 1
    with pytest.raises(cuda_lib.WasteCudaError) as e:
        a.call()
    assert e.value.rc == cuda_lib.E_ARG and "workspace" in str(e.value)


def test_attn_library_stream(cuda_lib):
    """stream 0 is the library's own, which device_errors waits for."""
    a = attn_case(cuda_lib, "tree").put()
    torch.cuda.synchronize()
    cuda_lib.mla_tree_attn_dev(a.d)
    cuda_lib.device_errors()
    a.check()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,H,ctx", [("bf16", 32, 0), ("bf16", 32, 199), ("f16", 32, 0), ("f16", 64, 199),
                                         ("f32", 4, 0), ("f32", 4, 99)])
def test_attn_far_scores(cuda_lib, dtype, H, ctx, sign):
    """Scores far beyond what 32 bits resolve to a unit, of both signs. All rows
    seen are the same, so whatever the weights round to, o is that row: in 16
    bits exactly, since 200 sums' 2^-24 each are no half step of the type."""
    a = Attn(cuda_lib, 3, dtype, H, 512, 64, 64, [ctx], [1], None)
    big = 3e4 if dtype == "f16" else 1e17
    a.q[:] = big
    a.cache[:] = sign * big
    a.put().call()
    torch.cuda.synchronize()
    want = float(a.cache[0, 0, 0])
    assert bool(((a.go[0].double() - want).abs() <= (512 * E * abs(want) if dtype == "f32" else 0)).all())
    lse = float(a.q[0, 0, 0].double()) * want * 576 * a.scale
    assert bool(((a.gl[0].double() - lse).abs() <= 700 * E * abs(lse)).all())
    assert cuda_lib.device_errors() == 0


@pytest.mark.parametrize("name", ["tree", "f32_tree", "pages_5"])
def test_attn_decreasing_indptr(cuda_lib, name):
    """Token ranges that go backwards would overlap: reported, nothing written."""
    wb = cuda_lib
    a = attn_case(wb, name).put()
    ip = [0, 1] * len(a.kv)
    a.gi.copy_(dev(ip[:len(a.kv) + 1][::-1] if len(a.kv) % 2 else ip[:len(a.kv) + 1]))
    a.gi[0], a.gi[1] = 2, 1
    a.call()
    assert wb.device_errors() == wb.DERR_BAD_BLOCK
    assert bool((a.go == 7).all()) and bool((a.gl == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["chains", "unserved", "unserved_one"])
def test_attn_segments_without_keys(cuda_lib, name, dtype):
    """Several segments a CTA, some of them without keys (the units that a
    chain's closed count adds; requests that were not served), so that what one
    segment left under way meets the next one's queries."""
    if name == "chains":
        a = Attn(cuda_lib, 21, dtype, 16, 128, 32, 64, [309, 242, 320, 297, 33], [50, 95, 89, 36, 67])
    else:
        n = 300
        a = Attn(cuda_lib, 22, dtype, 32, 128, 32, 16, [(37 * r) % 90 for r in range(n)], [2 if name == "unserved" else 1] * n,
                 unserved=[r for r in range(n) if r % 3])
    ref = a.ref()
    a.put()
    for _ in range(3):
        a.go.fill_(7.0)
        a.call().check(ref)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H", [32, 64])
@pytest.mark.parametrize("unit", [23, 24, 25, 26, 27, 28])
def test_attn_coarse_scores(cuda_lib, unit, H, dtype):
    """Scores where 32 bits step by 1 to 32: the difference to the reference of
    the tiles before, and that reference, are not exact there, and a weight may
    not leave the type for it. Scores are exact: products of powers of two plus
    whole steps, 128 keys a score, each next score larger by 8 in units of log2
    (or the step). 160 requests of three tiles, so that a CTA has several in a row."""
    step = max(8, 2 ** (unit - 23))
    for first in range(1, 8):                        # steps from the power of two: odd and even last bits
        a = Attn(cuda_lib, 3, dtype, H, 128, 64, 64, [383] * 160, [1] * 160, None)
        a.table[:] = a.table[0]
        a.scale = float(np.float32(np.log(2.0)))     # units of log2 (to 2^-24)
        a.q[:] = 0
        a.q[:, :, 0], a.q[:, :, 1] = 2.0 ** 13, 1.0
        a.cache[:] = torch.randn(a.cache.shape, generator=torch.Generator().manual_seed(first)).to(a.cache.dtype)
        rows = torch.from_numpy(a.table[0]).long()
        flat = a.cache[rows].view(-1, a.D)
        flat[:, 0] = 2.0 ** (unit - 13)
        flat[:128, 1] = first * 2.0 ** max(0, unit - 23)
        flat[128:256, 1] = first * 2.0 ** max(0, unit - 23) + step
        flat[256:, 1] = first * 2.0 ** max(0, unit - 23) + 2 * step
        a.cache[rows] = flat.view(len(rows), a.page, a.D)
        a.put().call()
        torch.cuda.synchronize()
        # weights 2^-2step, 2^-step and 1, exact but for the scale's 2^-24 of 16
        w = torch.exp2(-float(step) * torch.tensor([2.0, 1.0, 0.0], dtype=torch.float64)).repeat_interleave(128)
        lat = flat[:, :128].double()
        want = (w @ lat) / w.sum()
        size = (w @ lat.abs()) / w.sum()
        tol = size * (2 * HALF[dtype] + 1e-5) + 2.0 ** -30
        got = a.go[:a.T].cpu().double()
        assert bool(((got - want).abs() <= tol).all()), first
    assert cuda_lib.device_errors() == 0


def test_plan_cut_at_T(cuda_lib):
    """More new tokens than rows, in the middle of a request: the request has
    the rows that are there, its length counts those, and a chain planned so
    sees its cached rows and itself, none of the rows that nobody wrote."""
    wb = cuda_lib
    ctx, q, page = [0, 5, 3], [3, 6, 2], 4
    a = Attn(wb, 6, "bf16", 32, 512, 64, page, ctx, [3, 2, 0], None, extra=0)
    pl = Plan(wb, ctx, q, [0, 2, 1], [[-1, -1, -1], [8, 9, -1], [7, -1, -1]], list(range(7)), 0, page, 1, None, extra=-6)
    wb.kv_plan_dev(pl.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_TREE
    assert pl.t["q_indptr"].tolist() == [0, 3, 5, 5]
    assert pl.t["kv_len"].tolist() == [3, 7, 3]
    assert pl.t["slot"].tolist() == [0, 1, 2, 9 * page + 1, 9 * page + 2]
    a.table, a.kv = np.asarray(pl.t["block_table"].cpu(), np.int64), [3, 7, 3]
    a.cache = torch.randn(10, page, a.D, generator=torch.Generator().manual_seed(1)).to(a.cache.dtype)
    a.n_blocks = 10
    a.put()
    a.d.block_table, a.d.kv_len, a.d.q_indptr = (p(pl.t[k]) for k in ("block_table", "kv_len", "q_indptr"))
    a.call().check()


@pytest.mark.parametrize("name", ["tree", "f32_tree", "pages_5", "ragged"])
def test_attn_token_ranges(cuda_lib, name):
    """Token ranges outside 0..T: reported, nothing written."""
    wb = cuda_lib
    a = attn_case(wb, name).put()
    for r, x in ((0, -1), (0, -2 ** 31), (-1, a.T + a.extra + 1), (-1, 2 ** 31 - 1), (1, 2 ** 31 - 1)):
        a.gi.copy_(dev(a.indptr))
        a.gi[r] = x
        a.call()
        assert wb.device_errors() == wb.DERR_BAD_BLOCK
        assert bool((a.go == 7).all()) and bool((a.gl == 7).all())


@pytest.mark.parametrize("name", ["tree", "f32_tree"])
def test_attn_negative_length(cuda_lib, name):
    """A length below zero: reported, its tokens see nothing, the others' results stand."""
    wb = cuda_lib
    a = attn_case(wb, name)
    a.kv[0] = 0
    a.put()
    a.gk[0] = -5
    ref = a.ref()
    a.call()
    assert wb.device_errors() == wb.DERR_BAD_BLOCK
    a.check(ref)


@pytest.mark.parametrize("name", ["tree_wide", "f32_tree"])
def test_attn_mask_too_narrow(cuda_lib, name):
    """More new tokens than the mask's words have bits: reported, and the rows
    without a bit are seen by none."""
    wb = cuda_lib
    dtype, H, (kl, rope), page, ctx, q, tree = ATTN[name]
    a = Attn(wb, 3, dtype, H, kl, rope, page, [90, 5], [41, 3], 1)
    a.mask = np.ascontiguousarray(a.mask[:, :1])
    a.words = 1
    a.put()
    a.mask = np.concatenate([a.mask, np.zeros_like(a.mask)], 1)
    a.call()
    ref = a.ref()
    torch.cuda.synchronize()
    assert wb.device_errors() == wb.DERR_BAD_TREE
    a.check(ref)


# ---- logits --------------------------------------------------------------------------

class Logits:
    def __init__(self, wb, seed, dtype, V, q, hist_most, n_bias, pad=0, use=("hist", "draft", "tree", "bias", "allow", "rows"),
                 inplace=False, extra=1, prompt=True):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.wb, self.V, self.dtype, self.pad, self.extra = wb, V, dtype, pad, extra
        B, R = len(q), sum(q)
        self.indptr = [0]
        for n in q:
            self.indptr.append(self.indptr[-1] + n)
        self.R = R
        self.x = (torch.randn(R + extra, V + pad, generator=g) * 3).to(DT[dtype])
        few = max(2, V // 9)
        tok = lambda: rng.choice([rng.randrange(V), rng.randrange(few), V - 1, 0, -1, V, 2 ** 31 - 1, -2 ** 31])
        self.hist = [[tok() for _ in range(hist_most)] for _ in range(B)]
        self.hist_len = [rng.choice([0, 1, hist_most, rng.randrange(hist_most + 1)]) for _ in range(B)]
        self.prompt_len = [rng.choice([0, n, n // 2]) for n in self.hist_len] if prompt else None
        self.rep = [rng.choice([1.0, 1.3, 0.7]) for _ in range(B)]
        self.freq = [rng.choice([0.0, 0.25, -0.5]) for _ in range(B)]
        self.pres = [rng.choice([0.0, 0.6, -0.1]) for _ in range(B)]
        words = -(-max(1, max(q)) // 32)
        self.draft = [tok() for _ in range(R)] if "draft" in use else None
        self.tree = ancestors(parents(rng, q), q, words) if "tree" in use else None
        nb = [rng.choice([0, n_bias, rng.randrange(n_bias + 1)]) for _ in range(B)]
        # ids named twice: the last holds
        self.bias = [[(tok(), float(np.float32(rng.gauss(0, 2)))) for _ in range(n)] for n in nb] if "bias" in use else None
        aw = -(-V // 32)
        n_allow = R if "rows" not in use else max(1, R // 2)
        self.allow = np.random.default_rng(seed).integers(0, 1 << 32, (n_allow, aw), dtype=np.uint32) if "allow" in use else None
        if self.allow is not None:
            self.allow[0] = 0                                       # a grammar that allows nothing
        self.allow_row = [rng.randrange(-1, n_allow) for _ in range(R)] if "rows" in use else None
        if not any(k in use for k in ("hist",)):
            self.hist = None
        self.gx = self.x.cuda()
        self.gy = self.gx if inplace else torch.full_like(self.gx, 7.0)
        t = self.t = dict(logits=self.gx, out=self.gy, q_indptr=dev(self.indptr), rep=dev(self.rep, torch.float32),
                          freq=dev(self.freq, torch.float32), pres=dev(self.pres, torch.float32))
        if self.hist is not None:
            t.update(hist=dev(self.hist).view(B, -1), hist_len=dev(self.hist_len))
            if prompt:
                t.update(prompt_len=dev(self.prompt_len))
        if self.draft is not None:
            t["draft"] = dev(self.draft)
        if self.tree is not None:
            t["tree"] = u32(self.tree)
        if self.bias is not None:
            ptr = np.cumsum([0] + nb)
            t.update(bias_indptr=dev(ptr), bias_id=dev([v for b in self.bias for v, _ in b] + [0]),
                     bias_val=dev([x for b in self.bias for _, x in b] + [0], torch.float32))
        if self.allow is not None:
            t["allow"] = u32(self.allow)
            if self.allow_row is not None:
                t["allow_row"] = dev(self.allow_row)
        self.d = wb.LogitsAdjust(B=B, R=R + extra, V=V, dtype=CODE[dtype], tree_words=words, allow_words=aw,
                                 n_allow=n_allow, hist_stride=hist_most, ld=V + pad, ld_out=V + pad,
                                 **{k: p(v) for k, v in t.items()})

    def check(self):
        torch.cuda.synchronize()
        V = self.V
        x = self.x[:self.R, :V].double()
        ref = O.logits(x, self.indptr, self.hist, self.hist_len, self.prompt_len, self.rep, self.freq, self.pres,
                       self.draft, self.tree, self.bias, self.allow, self.allow_row)
        got = self.gy.cpu()
        rest = self.x if self.gy is self.gx else torch.full_like(self.x, 7.0)
        assert torch.equal(got[self.R:], rest[self.R:]) and torch.equal(got[:, V:], rest[:, V:])
        got = got[:self.R, :V].double()
        assert torch.equal(torch.isinf(got), torch.isinf(ref))
        fin = ~torch.isinf(ref)
        # five 32-bit roundings (parameters are floats: their own 2^-24), each of a value no larger
        # than the logit's share, the counted penalty's or the bias'
        n = len(self.hist[0]) + max(self.indptr) if self.hist is not None else max(self.indptr)
        size = x.abs() * 1.5 + 0.5 * n + 0.6 + 12
        tol = (ref.abs() * HALF[self.dtype] + 8 * E * size + TINY[self.dtype])[fin]
        d = (got - ref).abs()[fin]
        assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,q,hist,bias,pad", [
    (1, [1], 1, 1, 0), (33, [1, 1, 0, 2], 7, 5, 0), (1000, [3, 1, 5], 200, 40, 24), (1027, [2, 2], 90, 10, 0),
    (9001, [1] * 5, 600, 300, 3), (20000, [40, 1], 300, 20, 0)])
def test_logits(cuda_lib, dtype, V, q, hist, bias, pad):
    c = Logits(cuda_lib, V + len(q), dtype, V, q, hist, bias, pad)
    cuda_lib.logits_adjust_dev(c.d, stream())
    c.check()


@pytest.mark.parametrize("use", [(), ("hist",), ("draft",), ("hist", "draft", "tree"), ("bias",), ("allow",), ("allow", "rows"),
                                 ("hist", "bias", "allow")])
@pytest.mark.parametrize("inplace", [False, True])
def test_logits_parts(cuda_lib, use, inplace):
    c = Logits(cuda_lib, 17, "f32", 777, [2, 0, 3], 60, 12, use=use, inplace=inplace, extra=0, prompt="bias" not in use)
    for k in ("rep", "freq", "pres"):
        if not use:
            setattr(c.d, k, None)
    cuda_lib.logits_adjust_dev(c.d, stream())
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_many_named(cuda_lib, dtype):
    """More named ids in a slice than are taken at once, and more drafted ones
    than are listed."""
    c = Logits(cuda_lib, 12, dtype, 30000, [1, 300], 9000, 700)
    rng = random.Random(1)
    for r in range(2):
        c.hist[r] = rng.sample(range(30000), 9000)
        c.hist_len[r], c.prompt_len[r] = 9000, 4000
    c.draft[1:] = [rng.randrange(2000) for _ in range(300)]
    for k in ("hist", "hist_len", "prompt_len", "draft"):
        c.t[k].copy_(dev(getattr(c, k)).view(c.t[k].shape))
    cuda_lib.logits_adjust_dev(c.d, stream())
    rows = [0, 1, 2, 150, 300]
    got = c.gy.clone()
    torch.cuda.synchronize()
    # the definition goes row by row: a few of the rows
    x = c.x[:c.R, :c.V].double()
    ref = O.logits(x, c.indptr, c.hist, c.hist_len, c.prompt_len, c.rep, c.freq, c.pres, c.draft, c.tree, c.bias, c.allow,
                   c.allow_row, only=rows)
    for t in rows:
        fin = ~torch.isinf(ref[t])
        g = got[t, :c.V].cpu().double()
        assert torch.equal(torch.isinf(g), ~fin)
        size = x[t].abs() * 1.5 + 0.5 * 310 + 0.6 + 12
        tol = ref[t].abs() * HALF[dtype] + 8 * E * size + TINY[dtype]
        assert bool(((g - ref[t]).abs() <= tol)[fin].all())


@pytest.mark.parametrize("n", [4095, 4097, 8191, 8192, 8193, 10000])
@pytest.mark.parametrize("where", ["dense", "dense_end", "spread"])
def test_logits_named_pieces(cuda_lib, n, where):
    """As many named ids in a slice as are taken at once, one fewer and more:
    side by side at either end, or all over it. Values and penalties are whole
    numbers, so the results are exact."""
    wb, V = cuda_lib, 40000
    ids = {"dense": range(n), "dense_end": range(V - n, V), "spread": [i * 4 + i % 3 for i in range(n)]}[where]
    hist = random.Random(n).sample(list(ids), n)
    hist += hist[:50]
    x = torch.arange(V, dtype=torch.float32).view(1, V).repeat(64, 1)
    y = torch.full_like(x, 7.0).cuda()
    # rows of one request, so that the slices are wide
    t = dict(logits=x.cuda(), q_indptr=dev([0, 64]), hist=dev(hist), hist_len=dev([len(hist)]),
             freq=dev([2.0], torch.float32), pres=dev([1.0], torch.float32))
    for B in (1, 64):
        if B == 64:                                              # and a row a request
            t.update(q_indptr=dev(range(65)), hist=dev(hist * 64), hist_len=dev([len(hist)] * 64),
                     freq=dev([2.0] * 64, torch.float32), pres=dev([1.0] * 64, torch.float32))
        wb.logits_adjust_dev(wb.LogitsAdjust(B=B, R=64, V=V, dtype=wb.F32, hist_stride=len(hist), ld=V, ld_out=V, out=p(y),
                                             **{k: p(v) for k, v in t.items()}), stream())
        want = x[0].clone()
        want[hist[:n]] -= 3
        want[hist[:50]] -= 2
        assert torch.equal(y.cpu(), want.expand(64, V)), B
        y.fill_(7.0)
    assert wb.device_errors() == 0


def test_logits_mask_out_of_range(cuda_lib):
    wb = cuda_lib
    c = Logits(wb, 3, "f32", 500, [1, 1], 4, 2, use=("allow", "rows"), extra=0)
    c.t["allow_row"].copy_(dev([c.d.n_allow, 0]))
    wb.logits_adjust_dev(c.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_MASK
    assert bool(torch.isfinite(c.gy[0]).all()) and bool(torch.isinf(c.gy[1]).all())


def test_logits_row_per_request(cuda_lib):
    """Without q_indptr, row r is request r's."""
    c = Logits(cuda_lib, 4, "bf16", 5000, [1] * 6, 100, 9, extra=0)
    c.d.q_indptr = None
    cuda_lib.logits_adjust_dev(c.d, stream())
    c.check()


def test_logits_not_numbers(cuda_lib):
    """NaN and infinities pass through where they are allowed and become
    -infinity where they are not."""
    wb = cuda_lib
    V = 256
    for dtype in ("f32", "bf16"):
        x = torch.randn(1, V).to(DT[dtype])
        x[0, ::7], x[0, 1::7], x[0, 2::7] = float("nan"), float("inf"), float("-inf")
        allow = np.zeros((1, V // 32), np.uint32)
        allow[0, :4] = 0xFFFFFFFF
        gx, ga = x.cuda(), u32(allow)
        y = torch.empty_like(gx)
        wb.logits_adjust_dev(wb.LogitsAdjust(B=1, R=1, V=V, dtype=CODE[dtype], allow_words=8, n_allow=1, ld=V, ld_out=V,
                                             logits=p(gx), out=p(y), allow=p(ga)), stream())
        y = y.cpu()
        assert torch.equal(y[0, :128].float().nan_to_num(5, 6, 7), x[0, :128].float().nan_to_num(5, 6, 7))
        assert bool((y[0, 128:] == float("-inf")).all())


def test_logits_too_many_drafts(cuda_lib):
    """A request of more rows than drafts are followed for: reported, its rows
    as without drafts, the other request's with them."""
    wb, n = cuda_lib, 4097
    draft = [t % 60 for t in range(n + 2)]
    x = torch.ones(n + 2, 64)
    y = torch.full_like(x, 7.0).cuda()
    t = dict(logits=x.cuda(), q_indptr=dev([0, n, n + 2]), draft=dev(draft), freq=dev([0.5, 0.5], torch.float32))
    wb.logits_adjust_dev(wb.LogitsAdjust(B=2, R=n + 2, V=64, dtype=wb.F32, tree_words=0, ld=64, ld_out=64, out=p(y),
                                         **{k: p(v) for k, v in t.items()}), stream())
    assert wb.device_errors() == wb.DERR_BAD_TREE
    want = torch.ones(n + 2, 64)
    for row in (n, n + 1):
        for k in range(n, row + 1):
            want[row, draft[k]] -= 0.5
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("ptr", [[0, 5, 2, 6], [3, 1, 1, 1], [0, 2, 4, 12], [-1, 2, 4, 5], [0, 2 ** 31 - 1, 3, 6], [0, 4, 5, -2 ** 31]])
def test_logits_row_ranges(cuda_lib, ptr, inplace):
    """Ranges of rows that go backwards or leave 0..R: reported, nothing written."""
    wb = cuda_lib
    c = Logits(wb, 5, "f32", 3001, [2, 2, 2], 20, 4, inplace=inplace)
    c.t["q_indptr"].copy_(dev(ptr))
    wb.logits_adjust_dev(c.d, stream())
    assert wb.device_errors() == wb.DERR_BAD_BLOCK
    assert torch.equal(c.gy.cpu(), c.x if inplace else torch.full_like(c.x, 7.0))


@pytest.mark.parametrize("n", [-1, 21])
def test_logits_history_length(cuda_lib, n):
    """A history's length outside its row is reported and held to it."""
    wb = cuda_lib
    c = Logits(wb, 6, "f32", 300, [1, 2], 20, 4)
    c.hist_len[1] = max(0, min(20, n))
    c.prompt_len[1] = 3
    c.t["hist_len"][1], c.t["prompt_len"][1] = n, 3
    wb.logits_adjust_dev(c.d, stream())
    c.check()
    assert wb.device_errors() == wb.DERR_BAD_BLOCK


def test_logits_tree_too_narrow(cuda_lib):
    """More nodes than the tree's words have bits: reported, the rest of the
    nodes on no branch."""
    wb = cuda_lib
    c = Logits(wb, 7, "f32", 300, [40, 3], 20, 4)
    c.tree = np.ascontiguousarray(c.tree[:, :1])
    c.t["tree"] = u32(c.tree)
    c.d.tree, c.d.tree_words = p(c.t["tree"]), 1
    c.tree = np.concatenate([c.tree, np.zeros_like(c.tree)], 1)
    wb.logits_adjust_dev(c.d, stream())
    c.check()
    assert wb.device_errors() == wb.DERR_BAD_TREE


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_step_together(cuda_lib, dtype):
    """Two steps as a server makes them: a prompt's chunk for every request,
    then a tree of drafts for each, planned, written, attended and turned into
    adjusted logits, all from one stream with nothing read back between."""
    wb = cuda_lib
    rng, g = random.Random(2), torch.Generator().manual_seed(2)
    B, H, kl, rope, page, cols, V = 3, 32, 512, 64, 16, 12, 2000
    D, dt = kl + rope, DT[dtype]
    pool = 30
    cache = torch.zeros(pool, page, D, dtype=dt, device="cuda")
    model = torch.randn(H * kl, V, generator=g) * (H * kl) ** -0.5
    gm = model.cuda()
    w = 1 + 0.1 * torch.randn(kl, generator=g)
    inv = 10000.0 ** (-torch.arange(0, rope, 2).float() / rope)
    free = list(range(pool))
    rng.shuffle(free)
    held, table, head, ctx = [0] * B, np.full((B, cols), -1), 0, [0] * B
    known = torch.zeros(pool * page, D, dtype=torch.float64)           # the cache as the definition has it
    keep = []
    for step, q in enumerate(([20, 1, 33], [6, 9, 4])):
        T = sum(q)
        par = parents(rng, q) if step else None
        pl = Plan(wb, ctx, q, held, table, free, head, page, 2, par, extra=0)
        x, qq = torch.randn(T, D, generator=g), (torch.randn(T, H, D, generator=g)).to(dt)
        draft = [rng.randrange(V) for _ in range(T)]
        hist = dev([[rng.randrange(V) for _ in range(40)] for _ in range(B)])
        rep = dev([1.2] * B, torch.float32)
        gx, gq, gw, gi, gd = x.cuda(), qq.cuda(), w.cuda(), inv.cuda(), dev(draft)
        o = torch.empty(T, H, kl, dtype=dt, device="cuda")
        lse = torch.empty(T, H, device="cuda")
        n = wb.mla_tree_ws_bytes(H, kl)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        out = torch.empty(T, V, device="cuda")
        hl = dev([40] * B)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            wb.kv_plan_dev(pl.d, stream())
            wb.mla_rows_dev(wb.MlaRows(T=T, kl=kl, rope=rope, x_dtype=0, dtype=CODE[dtype], x_stride=D, x=p(gx), norm_w=p(gw),
                                       inv_freq=p(gi), pos=p(pl.t["pos"]), slot=p(pl.t["slot"]), eps=1e-6, cache=p(cache),
                                       row_stride=D, n_rows=pool * page), stream())
            wb.mla_tree_attn_dev(wb.MlaTree(
                B=B, T=T, heads=H, kl=kl, rope=rope, dtype=CODE[dtype], page=page, max_blocks=cols, mask_words=2,
                n_blocks=pool, row_stride=D, q_token_stride=H * D, q_head_stride=D, o_token_stride=H * kl,
                o_head_stride=kl, q=p(gq), cache=p(cache), block_table=p(pl.t["block_table"]), kv_len=p(pl.t["kv_len"]),
                q_indptr=p(pl.t["q_indptr"]), mask=p(pl.t["mask"]), scale=0.07, o=p(o), lse=p(lse), ws=p(ws), ws_bytes=n),
                stream())
            raw = o.view(T, -1).float() @ gm
            wb.logits_adjust_dev(wb.LogitsAdjust(
                B=B, R=T, V=V, dtype=0, tree_words=2, hist_stride=40, ld=V, ld_out=V, logits=p(raw), out=p(out),
                q_indptr=p(pl.t["q_indptr"]), hist=p(hist), hist_len=p(hl), rep=p(rep), draft=p(gd),
                tree=p(pl.t["mask"])), stream())
        torch.cuda.synchronize()
        keep.append((gx, gq, ws, raw))
        ref = O.plan(ctx, q, held, table, free, head, page, T, 2, par, cols)
        pl.check(ref)
        vals = O.rows(x, w, inv, torch.tensor(ref["pos"]), 1e-6)
        known[ref["slot"]] = vals
        got = cache.view(-1, D).cpu().double()
        tol = vals.abs() * (HALF[dtype] + (kl / 2 + 8) * E) + TINY[dtype]
        tol[:, kl:] += 12 * E * x[:, kl:].double().abs().view(T, -1, 2).sum(2).repeat_interleave(2, 1)
        assert bool(((got[ref["slot"]] - vals).abs() <= tol).all())
        # the attention of what the cache holds, the logits of what the attention gave
        ro, rl, to, tl = O.attn(qq, cache.cpu(), ref["table"], ref["kv_len"], ref["q_indptr"], ref["mask"], 0.07, kl, page, dtype)
        assert bool(((o.cpu().double() - ro).abs() <= to).all())
        assert bool(((lse.cpu().double() - rl).abs() <= tl).all())
        adj = O.logits(raw.cpu().double(), ref["q_indptr"], hist.cpu().tolist(), [40] * B, None, [1.2] * B, None, None, draft,
                       ref["mask"], None, None, None)
        size = raw.cpu().double().abs() * 1.5
        assert bool(((out.cpu().double() - adj).abs() <= adj.abs() * HALF["f32"] + 8 * E * size + TINY["f32"]).all())
        held, table, head = ref["n_blocks"], ref["table"], ref["head"]
        ctx = [c + n for c, n in zip(ctx, q)] if step == 0 else ctx
    assert wb.device_errors() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_step_captured_with_fewer_tokens(cuda_lib, dtype):
    """A whole step captured at T rows and replayed with fewer tokens, then with
    T again: the rows behind the last token are no token's, whatever slots and
    latents an earlier step left there, so kept rows stay what they were."""
    wb = cuda_lib
    rng, g = random.Random(8), torch.Generator().manual_seed(8)
    B, H, kl, rope, page, cols, V, T = 3, 32, 512, 64, 4, 10, 300, 12
    D, dt, pool = kl + rope, DT[dtype], 26
    cache = torch.zeros(pool, page, D, dtype=dt, device="cuda")
    free = list(range(pool))
    rng.shuffle(free)
    held, table, head, ctx = [0] * B, np.full((B, cols), -1), 0, [0] * B
    pl = Plan(wb, ctx, [4] * B, held, table, free, head, page, 1, None, extra=0, inplace=True)
    w = 1 + 0.1 * torch.randn(kl, generator=g)
    inv = 10000.0 ** (-torch.arange(0, rope, 2).float() / rope)
    gx, gw, gi = torch.zeros(T, D, device="cuda"), w.cuda(), inv.cuda()
    gq = torch.zeros(T, H, D, dtype=dt, device="cuda")
    o, lse = torch.empty(T, H, kl, dtype=dt, device="cuda"), torch.empty(T, H, device="cuda")
    raw, out = torch.zeros(T, V, device="cuda"), torch.empty(T, V, device="cuda")
    freq, draft = dev([0.5] * B, torch.float32), dev([0] * T)
    n = wb.mla_tree_ws_bytes(H, kl)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    t = pl.t
    calls = [
        (wb.kv_plan_dev, pl.d),
        (wb.mla_rows_dev, wb.MlaRows(
            T=T, kl=kl, rope=rope, x_dtype=0, dtype=CODE[dtype], x_stride=D, x=p(gx), norm_w=p(gw), inv_freq=p(gi),
            pos=p(t["pos"]), slot=p(t["slot"]), eps=1e-6, cache=p(cache), row_stride=D, n_rows=pool * page,
            n_tokens=p(t["q_indptr"]) + 4 * B)),
        (wb.mla_tree_attn_dev, wb.MlaTree(
            B=B, T=T, heads=H, kl=kl, rope=rope, dtype=CODE[dtype], page=page, max_blocks=cols, mask_words=1, n_blocks=pool,
            row_stride=D, q_token_stride=H * D, q_head_stride=D, o_token_stride=H * kl, o_head_stride=kl, q=p(gq),
            cache=p(cache), block_table=p(t["block_table"]), kv_len=p(t["kv_len"]), q_indptr=p(t["q_indptr"]),
            mask=p(t["mask"]), scale=0.07, o=p(o), lse=p(lse), ws=p(ws), ws_bytes=n)),
        (wb.logits_adjust_dev, wb.LogitsAdjust(
            B=B, R=T, V=V, dtype=0, tree_words=1, ld=V, ld_out=V, logits=p(raw), out=p(out), q_indptr=p(t["q_indptr"]),
            freq=p(freq), draft=p(draft), tree=p(t["mask"])))]
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        for f, d in calls:
            f(d, stream())
    known = torch.zeros(pool * page, D, dtype=torch.float64)
    for q in ([4, 4, 4], [1, 0, 2], [0, 3, 0], [4, 4, 4], [0, 0, 0], [1, 1, 1]):
        n = sum(q)
        x, qq = torch.randn(T, D, generator=g), torch.randn(T, H, D, generator=g).to(dt)
        y, ids = torch.randn(T, V, generator=g), [rng.randrange(V) for _ in range(T)]
        gx.copy_(x), gq.copy_(qq), raw.copy_(y), draft.copy_(dev(ids))
        o.fill_(7.0), lse.fill_(7.0), out.fill_(7.0)
        t["ctx_len"].copy_(dev(ctx)), t["q_len"].copy_(dev(q))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = O.plan(ctx, q, held, table, free, head, page, T, 1, None, cols)
        vals = O.rows(x[:n], w, inv, torch.tensor(ref["pos"]), 1e-6)
        if n:
            known[ref["slot"]] = vals
        got = cache.view(-1, D).cpu().double()
        # a row's rotated pairs are bounded by the pair's size, no more than the row's largest twice
        tol = known.abs() * (HALF[dtype] + (kl / 2 + 8) * E) + TINY[dtype]
        tol[:, kl:] += 24 * E * known[:, kl:].abs().amax(1, keepdim=True)
        assert bool(((got - known).abs() <= tol).all()), q
        if n:
            ro, rl, to, tl = O.attn(qq[:n], cache.cpu(), ref["table"], ref["kv_len"], ref["q_indptr"], ref["mask"], 0.07, kl, page, dtype)
            assert bool(((o[:n].cpu().double() - ro).abs() <= to).all())
            assert bool(((lse[:n].cpu().double() - rl).abs() <= tl).all())
            adj = O.logits(y[:n].double(), ref["q_indptr"], None, None, None, None, [0.5] * B, None, ids, ref["mask"], None, None, None)
            assert bool(((out[:n].cpu().double() - adj).abs() <= (adj.abs() + 8 * y[:n].abs() + 8) * E).all())
        assert bool((o[n:] == 7).all()) and bool((lse[n:] == 7).all()) and bool((out[n:] == 7).all())
        held, table, head = ref["n_blocks"], ref["table"], ref["head"]
        ctx = [c + k for c, k in zip(ctx, q)]
    assert wb.device_errors() == 0


@pytest.mark.parametrize("there,bad", [(0, 0), (2, 0), (5, 0), (6, 1), (-1, 1)])
def test_rows_counted_on_device(cuda_lib, there, bad):
    """n_tokens rows are written, of T; outside 0..T it is reported, nothing written."""
    wb = cuda_lib
    x, w, c = torch.randn(5, 80).cuda(), torch.ones(64).cuda(), torch.zeros(6, 80).cuda()
    slot, n = dev([4, 1, 0, 3, 5], torch.int64), dev([there])
    wb.mla_rows_dev(wb.MlaRows(T=5, kl=64, rope=16, x_dtype=0, dtype=0, x_stride=80, x=p(x), norm_w=p(w), slot=p(slot),
                               eps=1e-6, cache=p(c), row_stride=80, n_rows=6, n_tokens=p(n)), stream())
    assert wb.device_errors() == (wb.DERR_BAD_BLOCK if bad else 0)
    wrote = (c != 0).any(1).tolist()
    assert [r for r in range(6) if wrote[r]] == sorted([4, 1, 0, 3, 5][:0 if bad else there])


def test_errors_raised_while_read(cuda_lib):
    """A bit raised on one stream while another kind is read and cleared is still
    there afterwards: every step's two faults are reported, by then at the latest."""
    wb = cuda_lib
    x, w, c, slot = torch.randn(1, 80).cuda(), torch.ones(64).cuda(), torch.zeros(1, 80).cuda(), dev([1], torch.int64)
    rows = wb.MlaRows(T=1, kl=64, rope=16, x_dtype=0, dtype=0, x_stride=80, x=p(x), norm_w=p(w), slot=p(slot), eps=1e-6,
                      cache=p(c), row_stride=80, n_rows=1)
    y, a, row = torch.randn(1, 32).cuda(), u32([[1]]), dev([1])
    adj = wb.LogitsAdjust(B=1, R=1, V=32, dtype=0, allow_words=1, n_allow=1, ld=32, ld_out=32, logits=p(y), out=p(y),
                          allow=p(a), allow_row=p(row))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for k in range(300):
        wb.mla_rows_dev(rows, s1.cuda_stream)
        s1.synchronize()
        wb.logits_adjust_dev(adj, s2.cuda_stream)
        got = wb.device_errors()
        s2.synchronize()
        got |= wb.device_errors()
        assert got == wb.DERR_BAD_BLOCK | wb.DERR_BAD_MASK, k
    assert wb.device_errors() == 0
