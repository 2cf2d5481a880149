"""Cases of the 4-bit head and the filtered sampler, with their plain forms.

Three operators of a decode step's LM head:

``sample``     one token per row of logits [rows, n] and its probability:
               temperature, min-p, top-k and top-p filters, then an inverse-CDF
               draw with a given uniform number per row
               (``flash_head.sampling.sample_logits``).
``w4``         logits [rows, vocab] of a head whose weight is held in 4 bits
               with a scale (and a zero point) per group of a row
               (``flash_head.w4.w4_logits``).
``w4_probes``  the same product for probed clusters only: logits [rows, p * cap]
               of each row's own clusters (``flash_head.w4.w4_block_sparse_logits``).

``run`` computes the plain forms (elementary torch operations, fp32 or fp64)
unless ``own`` is true; then it makes the calls a user makes.

A 4-bit weight is w = (q - zero) * scale: q in 0..15, two per byte (even column
in the low nibble), one scale per group of a row, zero = 8 without zero points.

A row of logits is sampled over its entries above -inf (NaN counts as masked),
ordered by falling logit, then rising column:
  1. min-p keeps the entries with p_i >= min_p * max p;
  2. top-k keeps the first k of them;
  3. top-p keeps the shortest prefix that holds at least top_p of their mass;
  4. the draw: M the kept mass, the first kept column (in column order) whose
     running mass exceeds u * M; its probability is its share of M.
A temperature of 0 takes the first entry of the order; a row without entries
gives -1 and probability 0. A filter is off at min_p 0, top_k 0, top_p 1.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_F = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one user's next token: 128K vocabulary, the usual chat settings
        {"name": "sample_1", "op": "sample", "rows": 1, "n": 128256, "dtype": "bf16",
         "filters": "chat", "masked": False, "ids": False},
        # a serving batch, every request with settings of its own (some greedy,
        # some without filters)
        {"name": "sample_64_mixed", "op": "sample", "rows": 64, "n": 128256, "dtype": "bf16",
         "filters": "mixed", "masked": False, "ids": False},
        # a full batch of float logits (after penalties), nucleus sampling
        {"name": "sample_256_topp_fp32", "op": "sample", "rows": 256, "n": 151936,
         "dtype": "fp32", "filters": "topp", "masked": False, "ids": False},
        # a full batch at a temperature alone: the whole vocabulary is kept
        {"name": "sample_256_plain", "op": "sample", "rows": 256, "n": 128256, "dtype": "bf16",
         "filters": "none", "masked": False, "ids": False},
        # candidate set of a FlashHead step: 256 probes of 16 tokens and 15
        # special tokens, columns mapped to vocabulary ids
        {"name": "sample_128_candidates", "op": "sample", "rows": 128, "n": 4111,
         "dtype": "bf16", "filters": "mixed", "masked": False, "ids": True},
        # grammar-constrained decoding: most of an odd-sized vocabulary masked
        {"name": "sample_24_masked", "op": "sample", "rows": 24, "n": 32003, "dtype": "fp16",
         "filters": "minp", "masked": True, "ids": False},
        # one row through the 4-bit 2048 x 128256 head: the decode step itself
        {"name": "w4_1x2048", "op": "w4", "rows": 1, "vocab": 128256, "hidden": 2048,
         "group": 128, "zeros": False, "dtype": "bf16"},
        # a small batch on a 4096-wide head, zero points, groups of 64
        {"name": "w4_8x4096", "op": "w4", "rows": 8, "vocab": 128256, "hidden": 4096,
         "group": 64, "zeros": True, "dtype": "fp16"},
        # a serving batch on the 1536 x 151936 head
        {"name": "w4_64x1536", "op": "w4", "rows": 64, "vocab": 151936, "hidden": 1536,
         "group": 128, "zeros": False, "dtype": "bf16"},
        # a full batch (the dense branch of a batched call)
        {"name": "w4_256x2048", "op": "w4", "rows": 256, "vocab": 128256, "hidden": 2048,
         "group": 128, "zeros": True, "dtype": "bf16"},
        # stage 2 of one decode row: 256 of 8016 clusters of 16 tokens
        {"name": "w4_probes_1", "op": "w4_probes", "rows": 1, "clusters": 8016, "cap": 16,
         "probes": 256, "hidden": 2048, "group": 128, "zeros": False, "dtype": "bf16"},
        # stage 2 of a small batch on the 4096-wide head
        {"name": "w4_probes_12", "op": "w4_probes", "rows": 12, "clusters": 8016, "cap": 16,
         "probes": 256, "hidden": 4096, "group": 64, "zeros": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "w4", "w4_probes"])
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 256), "n": _log(rng, 1000, 151936),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "filters": rng.choice(["chat", "mixed", "topp", "none", "minp"]),
                "masked": rng.random() < 0.3, "ids": rng.random() < 0.3}
    group = rng.choice([32, 64, 128])
    case = {"op": op, "group": group, "zeros": rng.random() < 0.5,
            "dtype": rng.choice(["bf16", "fp16"])}
    hidden = max(1, round(_log(rng, 512, 8192) / group)) * group
    if op == "w4":
        vocab = min(_log(rng, 2000, 151936), 128256 * 8192 // hidden)
        most = 256 * 128256 * 2048 // (vocab * hidden)
        return {**case, "rows": min(_log(rng, 1, 256), most), "vocab": vocab, "hidden": hidden}
    cap = rng.choice([4, 8, 16, 16, 16, 24])
    clusters = _log(rng, 500, 9496)
    return {**case, "rows": _log(rng, 1, 16), "clusters": clusters, "cap": cap,
            "probes": min(clusters, _log(rng, 16, 512)), "hidden": hidden}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _logits(case, g):
    """Logits as a decode step meets them: a broad bulk and, on top, some
    tokens whose logits fall with the logarithm of their rank; rows range from
    undecided to nearly certain."""
    B, n = case["rows"], case["n"]
    x = torch.randn(B, n, generator=g, device="cuda") * 2.0
    top = min(n, 200)
    at = torch.randint(0, n, (B, top), generator=g, device="cuda")
    head = 11.0 + 9.0 * torch.rand(B, 1, generator=g, device="cuda")
    rank = torch.arange(1, top + 1, device="cuda").float()
    val = head - 1.7 * torch.log(rank) + torch.randn(B, top, generator=g, device="cuda")
    x.scatter_reduce_(1, at, val, "amax")
    x = x.to(_F[case["dtype"]])
    if case["masked"]:
        share = torch.rand(B, 1, generator=g, device="cuda") * 0.9 + 0.099
        gone = torch.rand(B, n, generator=g, device="cuda") < share
        x.masked_fill_(gone, float("-inf"))
    return x


def _filters(case, g):
    B, kind = case["rows"], case["filters"]
    r = torch.rand(4, B, generator=g, device="cuda")
    t = torch.full((B,), 0.8, device="cuda")
    k = torch.zeros(B, dtype=torch.int32, device="cuda")
    p = torch.ones(B, device="cuda")
    m = torch.zeros(B, device="cuda")
    if kind == "none":
        return {"temperature": t + 0.2}
    if kind == "chat":
        return {"temperature": t, "top_k": k + 50, "top_p": p * 0.95, "min_p": m + 0.02}
    if kind == "topp":
        return {"temperature": t, "top_p": p * 0.9}
    if kind == "minp":
        return {"temperature": t + 0.2, "min_p": m + 0.05}
    t = torch.where(r[0] < 0.125, torch.zeros_like(t), 0.3 + r[0])
    k = torch.where(r[1] < 0.5, k, (1 + r[1] * 400).to(torch.int32))
    p = torch.where(r[2] < 0.4, p, 0.5 + r[2] * 0.49)
    m = torch.where(r[3] < 0.6, m, r[3] * 0.1)
    return {"temperature": t, "top_k": k, "top_p": p, "min_p": m}


def _quantized(vocab, case, g):
    """Nibbles [vocab, hidden / 2] uint8, scales [vocab, groups], zero points
    [vocab, groups] uint8 or None, as a 4-bit checkpoint holds them."""
    D, G = case["hidden"], case["hidden"] // case["group"]
    dt = _F[case["dtype"]]
    q = torch.empty(vocab, D // 2, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // D)
    for lo in range(0, vocab, step):
        hi = min(vocab, lo + step)
        v = (torch.randn(hi - lo, D, generator=g, device="cuda") * 2.7 + 8.0).round_().clamp_(0, 15)
        v = v.to(torch.uint8)
        q[lo:hi] = v[:, 0::2] | (v[:, 1::2] << 4)
    s = ((0.75 + 0.5 * torch.rand(vocab, G, generator=g, device="cuda")) * 0.0077).to(dt)
    z = None
    if case["zeros"]:
        z = torch.randint(6, 11, (vocab, G), generator=g, device="cuda").to(torch.uint8)
    return q, s, z


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "sample":
        st = {"logits": _logits(case, g), **_filters(case, g)}
        st["uniforms"] = torch.rand(case["rows"], generator=g, device="cuda", dtype=torch.float64)
        if case["ids"]:
            st["ids"] = torch.randint(0, 151936, (case["rows"], case["n"]), generator=g,
                                      device="cuda", dtype=torch.int32)
        return st
    vocab = case["vocab"] if case["op"] == "w4" else case["clusters"] * case["cap"]
    q, s, z = _quantized(vocab, case, g)
    h = (torch.randn(case["rows"], case["hidden"], generator=g, device="cuda") * 0.5)
    st = {"q": q, "scales": s, "zeros": z, "h": h.to(_F[case["dtype"]])}
    if case["op"] == "w4_probes":
        r = torch.rand(case["rows"], case["clusters"], generator=g, device="cuda")
        st["ci"] = r.topk(case["probes"], dim=1).indices.sort(dim=1).values
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own and case["op"] != "sample":
        _package()
        from flash_head.w4 import W4Weight
        st["weight"] = W4Weight.from_quantized(st.pop("q"), st.pop("scales"), st.pop("zeros"))
    return st


def _package():
    path = os.path.join(os.getcwd(), "flash-head_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_sample(st):
    x = st["logits"].float()
    B, n = x.shape
    x = x.masked_fill(x.isnan(), float("-inf"))
    T = st["temperature"].double().view(B, 1)
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = xs[:, :1].double()
    w = torch.exp((xs.double() - top) / T.clamp_min(1e-30))
    keep = xs > float("-inf")
    if "min_p" in st:
        keep &= w >= st["min_p"].double().view(B, 1)
    at = torch.arange(n, device=x.device).view(1, n)
    if "top_k" in st:
        k = st["top_k"].long().view(B, 1)
        keep &= (at < k) | (k <= 0)
    keep[:, :1] = xs[:, :1] > float("-inf")
    w = w * keep
    if "top_p" in st:
        p = st["top_p"].double().view(B, 1)
        run_mass = torch.cumsum(w, dim=1)
        before = torch.cat([torch.zeros_like(run_mass[:, :1]), run_mass[:, :-1]], dim=1)
        w = w * ((before < p * run_mass[:, -1:]) | (p >= 1) | (at == 0))
    w = torch.where((T <= 0) & (at > 0), torch.zeros_like(w), w)
    w = torch.zeros_like(w).scatter_(1, order, w)
    cum = torch.cumsum(w, dim=1)
    col = (cum <= st["uniforms"].view(B, 1) * cum[:, -1:]).sum(dim=1, keepdim=True)
    col = col.clamp_max(n - 1)
    prob = (w.gather(1, col) / cum[:, -1:]).float().view(B)
    out = (st["ids"].gather(1, col).long() if "ids" in st else col).view(B)
    none = xs[:, 0] == float("-inf")
    return out.masked_fill(none, -1), prob.masked_fill(none, 0.0)


def _plain_weight(q, s, z):
    V, D = q.shape[0], q.shape[1] * 2
    w = torch.stack([q & 15, q >> 4], dim=2).view(V, s.shape[1], -1).float()
    w = w - (8.0 if z is None else z.float().unsqueeze(2))
    return (w * s.float().unsqueeze(2)).view(V, D)


def run(st):
    case = st["case"]
    if case["op"] == "sample":
        if own:
            _package()
            from flash_head.sampling import sample_logits
            names = ("temperature", "top_k", "top_p", "min_p", "ids")
            return sample_logits(st["logits"], st["uniforms"], return_prob=True,
                                 **{k: st[k] for k in names if k in st})
        return _plain_sample(st)
    h = st["h"]
    if own:
        from flash_head.w4 import w4_block_sparse_logits, w4_logits
        if case["op"] == "w4":
            return w4_logits(h, st["weight"])
        return w4_block_sparse_logits(h, st["weight"], st["ci"], case["clusters"], case["cap"])
    if case["op"] == "w4":
        return (h.float() @ _plain_weight(st["q"], st["scales"], st["zeros"]).t()).to(h.dtype)
    cap, ci = case["cap"], st["ci"]
    rows = (ci.unsqueeze(2) * cap + torch.arange(cap, device=ci.device)).view(-1)
    z = None if st["zeros"] is None else st["zeros"][rows]
    w = _plain_weight(st["q"][rows], st["scales"][rows], z).view(h.shape[0], -1, h.shape[1])
    return (w * h.float().unsqueeze(1)).sum(dim=2).to(h.dtype)


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    B = case["rows"]
    if case["op"] == "sample":
        filters = {"none": 1, "chat": 4, "topp": 2, "minp": 2, "mixed": 4}[case["filters"]]
        # of the column ids only the drawn ones are needed
        moved = B * (case["n"] * size + 4 * filters + 8 + 12 + (4 if case["ids"] else 0))
        return {"bytes": moved, "flops": 4 * B * case["n"]}
    D = case["hidden"]
    row = D // 2 + D // case["group"] * (2 + (1 if case["zeros"] else 0))
    if case["op"] == "w4":
        V = case["vocab"]
        return {"bytes": V * row + B * D * 2 + B * V * 2, "flops": 2 * B * V * D}
    K, p, cap = case["clusters"], case["probes"], case["cap"]
    # rows choose their clusters independently: the expected number of distinct ones
    distinct = K * (1.0 - (1.0 - p / K) ** B)
    return {"bytes": int(distinct * cap * row) + B * (D * 2 + p * 8 + p * cap * 2),
            "flops": 2 * B * p * cap * D}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_row(x, u, T, k, p, m):
    """The drawn column of one row (numpy) and its probability, or -1 and 0."""
    cols = np.flatnonzero(x > -np.inf)  # NaN compares false
    if cols.size == 0:
        return -1, 0.0
    order = cols[np.argsort(-x[cols], kind="stable")]
    if T <= 0:
        return int(order[0]), 1.0
    e = np.exp((x[order] - x[order[0]]) / T)
    count = order.size
    if m > 0:
        count = max(1, int(np.count_nonzero(e >= m)))
    if k > 0:
        count = min(count, k)
    if p < 1:
        mass = np.concatenate([[0.0], np.cumsum(e[:count])])
        count = max(1, int(np.searchsorted(mass[:count], p * mass[count], side="left")))
    by_column = np.argsort(order[:count])
    mass = np.cumsum(e[:count][by_column])
    j = min(int(np.searchsorted(mass, u * mass[-1], side="right")), count - 1)
    return int(order[:count][by_column[j]]), float(e[:count][by_column[j]] / mass[-1])


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "sample":
        B = case["rows"]
        x = st["logits"].float().cpu().numpy().astype(np.float64)
        u = st["uniforms"].cpu().numpy()

        def col(name, off):
            v = st[name].cpu().numpy() if name in st else np.full(B, off)
            return v.astype(np.float64)
        T, k, p, m = col("temperature", 1), col("top_k", 0), col("top_p", 1), col("min_p", 0)
        rows = [_exact_row(x[r], u[r], T[r], int(k[r]), p[r], m[r]) for r in range(B)]
        got = np.array([r[0] for r in rows], dtype=np.int64)
        if "ids" in st:
            ids = st["ids"].cpu().numpy()
            got = np.where(got < 0, -1, ids[np.arange(B), np.maximum(got, 0)])
        return torch.from_numpy(got).cuda(), torch.tensor([r[1] for r in rows],
                                                          dtype=torch.float64, device="cuda")
    h = st["h"].double()
    q, s, z = st["q"], st["scales"], st["zeros"]
    V, G, group = q.shape[0], s.shape[1], case["group"]

    def part(rows_q, rows_s, rows_z, hh):
        # per group: scale * (sum of q * h  -  zero * sum of h)
        hg = hh.view(hh.shape[0], G, group)
        v = torch.empty(rows_q.shape[0], 2 * rows_q.shape[1], dtype=torch.float64, device="cuda")
        v[:, 0::2] = (rows_q % 16).double()
        v[:, 1::2] = (rows_q // 16).double()
        dots = torch.einsum("bgk,vgk->bvg", hg, v.view(-1, G, group))
        zero = 8.0 if rows_z is None else rows_z.double()
        return ((dots - hg.sum(2).unsqueeze(1) * zero) * rows_s.double()).sum(2)

    if case["op"] == "w4":
        step = max(1, (1 << 27) // max(case["hidden"], G * case["rows"]))
        outs = [part(q[lo:lo + step], s[lo:lo + step], None if z is None else z[lo:lo + step], h)
                for lo in range(0, V, step)]
        return torch.cat(outs, dim=1)
    outs = []
    for r in range(case["rows"]):
        rows = (st["ci"][r].unsqueeze(1) * case["cap"]
                + torch.arange(case["cap"], device="cuda")).view(-1)
        outs.append(part(q[rows], s[rows], None if z is None else z[rows], h[r:r + 1]))
    return torch.cat(outs, dim=0)
