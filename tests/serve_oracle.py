"""Plain 64-bit forms of the serving step's operators, for its tests: loops
over requests, tokens and ids, written from the definitions in
include/waste_cuda.h."""
import numpy as np
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
#: half a step of the type, relative to the value
HALF = {k: torch.finfo(t).eps / 2 for k, t in DT.items()}
#: half of the type's smallest step (its subnormals')
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def plan(ctx, q, held, table, free, head, page, T, words, parent, max_blocks, masked=True):
    """kv_plan: a dict of its outputs (numpy), the table updated in a copy."""
    B = len(ctx)
    table, held = np.array(table), list(held)
    indptr, pos, slot, mask = [0], [], [], []
    kv, at, before, short, bad = [], head, 0, 0, 0
    avail = max(0, len(free) - head)
    for r in range(B):
        blocks = -(-(ctx[r] + q[r]) // page)
        ok = blocks <= max_blocks and not (masked and q[r] > 32 * words)
        need = max(0, blocks - held[r]) if ok else 0
        served = ok and (need == 0 or before + need <= avail)
        before += need
        if served:
            for j in range(need):
                table[r, held[r] + j] = free[at + j]
            at += need
            held[r] += need
        kv.append(ctx[r] + q[r] if served else 0)
        t0 = indptr[-1]
        anc = []
        for i in range(q[r]):
            p = i - 1 if parent is None else parent[t0 + i]
            anc.append((anc[p] if p >= 0 else []) + [i])
            pos.append(ctx[r] + len(anc[i]) - 1)
            n = ctx[r] + i
            slot.append(int(table[r, n // page]) * page + n % page if served else -1)
            row = [0] * words
            for j in anc[i]:
                if j < 32 * words:
                    row[j // 32] |= 1 << (j % 32)
            mask.append(row)
        indptr.append(t0 + q[r])
    short = max(0, before - avail)
    return {"table": table, "n_blocks": held, "head": at, "q_indptr": [min(x, T) for x in indptr], "kv_len": kv,
            "pos": pos[:T], "slot": slot[:T], "mask": np.array(mask, np.uint32).reshape(-1, words)[:T], "short": short}


def rows(x, w, inv_freq, pos, eps):
    """mla_rows' values [T][kl + rope] in 64 bits."""
    x, kl = x.double(), w.numel()
    lat = x[:, :kl]
    lat = lat / torch.sqrt((lat ** 2).mean(1, keepdim=True) + float(np.float32(eps))) * w.double()
    r = x[:, kl:].clone()
    if inv_freq is not None:
        a = pos.double()[:, None] * inv_freq.double()[None, :]
        e, o = x[:, kl::2], x[:, kl + 1::2]
        r[:, 0::2] = e * a.cos() - o * a.sin()
        r[:, 1::2] = e * a.sin() + o * a.cos()
    return torch.cat([lat, r], 1)


def attn(q, cache, table, kv_len, indptr, mask, scale, kl, page, dtype):
    """(o, lse, tolerance of o, tolerance of lse) in 64 bits. q [T][H][D], cache
    [blocks][page][D] on the CPU, mask [T][words] (numpy, uint32) or None.

    The tolerances, for a row of n seen keys, with e = 2^-24:
      score    |ds| <= (D + 3) e scale sum|q c| =: g, and the exponential's argument is off by 2 e
               (|s| + |max|) more and its value by 4 e: a weight is off by a share of
               2 (g + 2 e (|s| + |max|)) + 4 e =: h
      weights  rounded to a 16-bit type: half a step, u (and at most the type's smallest half step)
      products sum of n terms, in parts and joined: (n + 32) e sum w|c|
      result   sum w|c| (h + u + (n + 32) e), the normaliser's own h + (n + 32) e, rounded: u |o|
      lse      g + h + (n + 32) e + 4 e |lse|
    """
    T, H, D = q.shape
    o = torch.zeros(T, H, kl, dtype=torch.float64)
    lse = torch.full((T, H), -np.inf, dtype=torch.float64)
    to, tl = torch.zeros_like(o), torch.zeros_like(lse)
    e, u = 2.0 ** -24, HALF[dtype]
    uw = 0.0 if dtype == "f32" else u
    for r in range(len(kv_len)):
        a, b, n = indptr[r], indptr[r + 1], kv_len[r]
        if n < b - a:
            continue
        c = n - (b - a)
        ids = torch.as_tensor(table[r][:-(-n // page)]).long()
        lat = cache[ids].reshape(-1, D)[:n].double()
        for t in range(a, b):
            see = [p for p in range(n) if p < c or (p - c <= t - a if mask is None else
                                                    (int(mask[t][(p - c) // 32]) >> ((p - c) % 32)) & 1)]
            if not see:
                continue
            k = lat[see]
            qq = q[t].double()
            s = qq @ k.T * scale
            z = torch.logsumexp(s, 1)
            w = torch.exp(s - z[:, None])
            o[t] = w @ k[:, :kl]
            lse[t] = z
            m = len(see)
            g = (D + 3) * e * abs(scale) * (qq.abs() @ k.abs().T).amax(1)
            h = 2 * (g + 4 * e * s.abs().amax(1)) + 4 * e
            wv = w @ k[:, :kl].abs()
            to[t] = wv * (2 * h[:, None] + uw + 2 * (m + 32) * e) + u * o[t].abs() + TINY[dtype] + \
                (m * 2.0 ** -25 * k[:, :kl].abs().amax(0)[None, :] if dtype == "f16" else 0.0) * 2.0 ** -8
            tl[t] = g + h + (m + 32) * e + 4 * e * z.abs()
    return o, lse, to, tl


def logits(x, indptr, hist, hist_len, prompt_len, rep, freq, pres, draft, tree, bias, allow, allow_row, only=None):
    """One row at a time: x [R][V] (64 bits); bias: per request a list of (id, value);
    only: the rows to do."""
    R, V = x.shape
    out = x.clone()
    for r in range(len(indptr) - 1):
        for t in range(indptr[r], indptr[r + 1]):
            if only is not None and t not in only:
                continue
            seen, n = torch.zeros(V, dtype=torch.bool), torch.zeros(V, dtype=torch.float64)
            if hist is not None:
                for i, v in enumerate(hist[r][:hist_len[r]]):
                    if 0 <= v < V:
                        seen[v] = True
                        n[v] += i >= (prompt_len[r] if prompt_len is not None else 0)
            if draft is not None:
                for j in range(indptr[r + 1] - indptr[r]):
                    on = j <= t - indptr[r] if tree is None else (int(tree[t][j // 32]) >> (j % 32)) & 1
                    v = draft[indptr[r] + j]
                    if on and 0 <= v < V:
                        seen[v] = True
                        n[v] += 1
            y = x[t]
            p = float(rep[r]) if rep is not None else 1.0
            y = torch.where(seen, torch.where(y > 0, y / p, y * p), y)
            y = y - (float(freq[r]) if freq is not None else 0.0) * n
            y = y - (float(pres[r]) if pres is not None else 0.0) * (n > 0)
            for v, val in dict(bias[r]).items() if bias is not None else ():
                if 0 <= v < V:
                    y[v] += val
            if allow is not None:
                a = allow_row[t] if allow_row is not None else t
                if a >= 0:
                    ok = torch.tensor([(int(allow[a][v // 32]) >> (v % 32)) & 1 for v in range(V)], dtype=torch.bool)
                    y = torch.where(ok, y, -torch.inf)
            out[t] = y
    return out
