"""What is measured of the operators that check drafted tokens over the int8 KV cache: attention of a tree of drafted
tokens (``tree_attn_i8``), the walk that accepts a path of it (``tree_accept``), the compaction of the cache to that path
(``kv_compact_i8``), token sampling (``sample_f32``) and the residual RMSNorm with int8 output (``add_rmsnorm_quant``).

``run`` computes an operator in its plain form with elementary torch operations or, where ``own`` is true, calls the
framework's entry point.
"""
import math
import random

import numpy as np
import torch

own = False

DIM = 128  # the head dimension of every int8 attention operator


def listed():
    return [
        # a chat of one user: four tokens drafted in a chain, every head with its own keys
        dict(name="tree_1x4_h32", op="tree", batch=1, drafts=4, heads_q=32, heads_kv=32, len=499, max_len=512, ragged=False, chain=True),
        # a served batch on one of eight shards: 8 query heads on one KV head, trees of 8, lengths all different
        dict(name="tree_64x8_4k", op="tree", batch=64, drafts=8, heads_q=8, heads_kv=1, len=4096, max_len=4160, ragged=True, chain=False),
        # two long documents with wide trees of 64
        dict(name="tree_2x64_16k", op="tree", batch=2, drafts=64, heads_q=64, heads_kv=8, len=16301, max_len=16384, ragged=False, chain=False),
        # one user's accepted rows in one layer's cache
        dict(name="compact_1x4", op="compact", layers=1, batch=1, drafts=4, heads_kv=32, max_len=512),
        # a served batch's accepted rows in every layer's cache at once
        dict(name="compact_16l_32x16", op="compact", layers=16, batch=32, drafts=16, heads_kv=8, max_len=512),
        # GPT-Neo's vocabulary, one user
        dict(name="sample_1x50257", op="sample", rows=1, n=50257, params="top_k", coarse=False),
        # a served batch whose requests all ask for something else; logits with few bits, so equal ones abound
        dict(name="sample_64x128000_mixed", op="sample", rows=64, n=128000, params="mixed", coarse=True),
        # a large batch with nucleus sampling
        dict(name="sample_256x128000_top_p", op="sample", rows=256, n=128000, params="top_p", coarse=False),
        # a decode step's rows
        dict(name="add_rms_64x8192", op="add_rms", rows=64, width=8192),
        # a prefill's rows
        dict(name="add_rms_16384x4096", op="add_rms", rows=16384, width=4096),
        # one user's tree, and a served batch's
        dict(name="accept_1x8", op="accept", batch=1, drafts=8),
        dict(name="accept_512x64", op="accept", batch=512, drafts=64),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "sample", "sample", "compact", "add_rms", "accept"])
    if op == "tree":
        heads_kv = rng.choice([1, 2, 8, 32])
        heads_q = heads_kv * rng.choice([1, 2, 4, 8, 16] if heads_kv < 32 else [1, 2])
        drafts = _spread(rng, 1, 64)
        length = _spread(rng, 1, 16000)
        batch = _spread(rng, 1, 64)
        while batch > 1 and (batch * heads_q * drafts * length > 2 * 64 * 64 * 16301 or batch * heads_kv * length > 64 * 4096):
            batch //= 2
        max_len = (length + drafts + 3) // 4 * 4 + 4 * rng.randrange(8)
        return dict(op="tree", batch=batch, drafts=drafts, heads_q=heads_q, heads_kv=heads_kv, len=length, max_len=max_len,
                    ragged=rng.random() < 0.5, chain=rng.random() < 0.3)
    if op == "compact":
        return dict(op="compact", layers=_spread(rng, 1, 16), batch=_spread(rng, 1, 32), drafts=_spread(rng, 1, 16),
                    heads_kv=rng.choice([1, 2, 4, 8]), max_len=4 * rng.randint(16, 128))
    if op == "sample":
        return dict(op="sample", rows=_spread(rng, 1, 256), n=_spread(rng, 2, 128000),
                    params=rng.choice(["top_k", "top_p", "min_p", "plain", "mixed"]), coarse=rng.random() < 0.5)
    if op == "add_rms":
        width = 32 * _spread(rng, 1, 512)
        return dict(op="add_rms", rows=_spread(rng, 1, 16384 * 4096 // max(width, 4096)), width=width)
    return dict(op="accept", batch=_spread(rng, 1, 512), drafts=_spread(rng, 1, 64))


def _lens(case):
    """The committed length of each sequence."""
    length, batch = case["len"], case["batch"]
    return [length - (b * 97) % (length // 2 + 1) if case["ragged"] else length for b in range(batch)]


def _draft_lens(case):
    """The drafted tokens of each sequence (a ragged batch has fewer for some)."""
    t, batch = case["drafts"], case["batch"]
    return [t - b % (t // 2 + 1) if case["ragged"] else t for b in range(batch)]


def _parents(r, batch, drafts):
    """Random trees: node 0 is the root (-1), every other node hangs under an earlier one."""
    p = np.floor(r.random_sample((batch, drafts)) * np.arange(drafts)).astype(np.int32)
    p[:, 0] = -1
    return p


def _rows8(gen, shape, std):
    """int8 rows of DIM with one fp32 scale each, as the cache holds them: scale = max|x| / 127."""
    x = torch.randn(shape + (DIM,), generator=gen, device="cuda") * std
    scale = x.abs().amax(-1) / 127.0
    return torch.round(x / scale[..., None]).clamp_(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 32))
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    s = {"case": case}
    if case["op"] == "tree":
        b, t, hq, hkv, m = (case[k] for k in ("batch", "drafts", "heads_q", "heads_kv", "max_len"))
        s["q8"], s["q_scale"] = _rows8(gen, (b, t, hq), 1.5)
        s["k"], s["k_scale"] = _rows8(gen, (b, hkv, m), 1.5)
        s["v"], s["v_scale"] = _rows8(gen, (b, hkv, m), 1.0)
        s["lens"] = dev(np.array(_lens(case), np.int32))
        s["draft_lens"] = dev(np.array(_draft_lens(case), np.int32)) if case["ragged"] else None
        s["parents"] = None if case["chain"] else dev(_parents(r, b, t))
        s["sm_scale"] = 1.0 / math.sqrt(DIM)
        s["out"] = torch.zeros((b, t, hq, DIM), device="cuda")  # a program's own buffer; rows past a sequence's drafts stay
    elif case["op"] == "compact":
        n, b, t, hkv, m = (case[k] for k in ("layers", "batch", "drafts", "heads_kv", "max_len"))
        shape = (n, b, hkv, m)
        for c in ("k", "v"):
            s[c] = torch.randint(-127, 128, shape + (DIM,), generator=gen, device="cuda", dtype=torch.int8)
            s[c + "_scale"] = torch.rand(shape, generator=gen, device="cuda") * 0.03 + 0.01
        lens = r.randint(0, m - t + 1, b).astype(np.int32)
        accepted = r.randint(1, t + 1, b).astype(np.int32)
        path = np.full((b, t), -1, np.int32)
        for i in range(b):  # node 0, then some of the others in order
            path[i, : accepted[i]] = np.concatenate([[0], np.sort(r.permutation(t - 1)[: accepted[i] - 1] + 1)])
        s["lens"], s["accepted"], s["path"] = dev(lens), dev(accepted), dev(path)
    elif case["op"] == "sample":
        rows, n = case["rows"], case["n"]
        x = torch.randn((rows, n), generator=gen, device="cuda") * 3.0
        if n > 64:  # a few likely tokens
            likely = torch.randint(0, n, (rows, 8), generator=gen, device="cuda")
            x += torch.zeros_like(x).scatter_(1, likely, 10.0)
        s["logits"] = x.bfloat16().float() if case["coarse"] else x
        s["u"] = torch.rand(rows, generator=gen, device="cuda")
        kind = case["params"]
        temperature = np.full(rows, 0.8, np.float32)
        top_k = top_p = min_p = None
        if kind in ("top_k", "mixed"):
            top_k = np.full(rows, 40, np.int32)
        if kind in ("top_p", "mixed"):
            top_p = np.full(rows, 0.9, np.float32)
        if kind in ("min_p", "mixed"):
            min_p = np.full(rows, 0.05, np.float32)
        if kind == "mixed":  # some greedy, some with one filter, some with all
            temperature = np.where(r.rand(rows) < 0.1, 0.0, r.uniform(0.4, 1.5, rows)).astype(np.float32)
            top_k = np.where(r.rand(rows) < 0.5, 0, r.randint(1, 1000, rows)).astype(np.int32)
            top_p = np.where(r.rand(rows) < 0.5, 1.0, r.uniform(0.5, 0.99, rows)).astype(np.float32)
            min_p = np.where(r.rand(rows) < 0.5, 0.0, r.uniform(0.01, 0.2, rows)).astype(np.float32)
        for key, a in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            s[key] = None if a is None else dev(a)
    elif case["op"] == "add_rms":
        rows, width = case["rows"], case["width"]
        s["x"] = torch.randn((rows, width), generator=gen, device="cuda")
        s["residual"] = torch.randn((rows, width), generator=gen, device="cuda") * 2.0
        s["gain"] = torch.rand(width, generator=gen, device="cuda") + 0.5
        s["eps"] = 1e-5
    else:
        b, t = case["batch"], case["drafts"]
        parents, tokens = _parents(r, b, t), r.randint(0, 50, (b, t)).astype(np.int32)
        chosen = r.randint(0, 50, (b, t)).astype(np.int32)
        for i in range(1, t):  # the model often chooses what was drafted
            hit = np.nonzero(r.rand(b) < 0.5)[0]
            chosen[hit, parents[hit, i]] = tokens[hit, i]
        s["parents"], s["tokens"], s["chosen"] = dev(parents), dev(tokens), dev(chosen)
    return s


def run(s):
    op = s["case"]["op"]
    return {"tree": _tree, "compact": _compact, "sample": _sample, "add_rms": _add_rms, "accept": _accept}[op](s)


def _ancestors(parents):
    """[b][t][t]: whether node j is an ancestor of node i or node i itself."""
    t = parents.shape[1]
    step = (parents[:, :, None] == torch.arange(t, device=parents.device)).float()
    return torch.linalg.matrix_power(step + torch.eye(t, device=parents.device), t) > 0


def _tree(s):
    if own:
        from reef_b200 import kernels as K
        return K.tree_attn_i8(s["q8"], s["q_scale"], s["k"], s["k_scale"], s["v"], s["v_scale"], s["lens"], parents=s["parents"],
                              draft_lens=s["draft_lens"], sm_scale=s["sm_scale"], out=s["out"])
    q8, k8, v8 = s["q8"], s["k"], s["v"]
    b, t, hq, _ = q8.shape
    hkv, m = k8.shape[1], k8.shape[2]
    g = hq // hkv
    q = (q8.float() * s["q_scale"][..., None]).view(b, t, hkv, g, DIM).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * t, DIM)
    k = k8.float() * s["k_scale"][..., None]
    scores = (q @ k.transpose(-1, -2)).view(b, hkv, g, t, m) * s["sm_scale"]
    lens = s["lens"].long()
    at = torch.arange(t, device=q8.device)
    parents = s["parents"] if s["parents"] is not None else (at - 1).to(torch.int32).expand(b, t)
    node = torch.arange(m, device=q8.device)[None] - lens[:, None]  # [b][m]: the drafted token at each row, negative before them
    inside = (node >= 0) & (node < t)
    drafted = _ancestors(parents).gather(2, node.clamp(0, t - 1)[:, None].expand(b, t, m))
    visible = (node < 0)[:, None] | (inside[:, None] & drafted)
    scores = scores.masked_fill(~visible[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = p.reshape(b, hkv, g * t, m) @ (v8.float() * s["v_scale"][..., None])
    out = out.view(b, hkv, g, t, DIM).permute(0, 3, 1, 2, 4).reshape(b, t, hq, DIM)
    if s["draft_lens"] is None:
        s["out"].copy_(out)
    else:
        s["out"].copy_(torch.where((at[None] < s["draft_lens"][:, None])[..., None, None], out, s["out"]))
    return s["out"]


def _compact(s):
    if own:
        from reef_b200 import kernels as K
        new_lens = K.kv_compact_i8(s["k"], s["k_scale"], s["v"], s["v_scale"], s["lens"], s["path"], s["accepted"])
    else:
        n, b, hkv, m, _ = s["k"].shape
        t = s["path"].shape[1]
        i = torch.arange(t, device=s["k"].device)
        live = i[None] < s["accepted"][:, None]
        lens = s["lens"].long()[:, None]
        to = (lens + i[None]).clamp(max=m - 1)
        source = torch.where(live, lens + s["path"], to)  # the rows past the accepted ones keep what they hold
        source, to = (x[None, :, None].expand(n, b, hkv, t) for x in (source, to))
        for c in ("k_scale", "v_scale"):
            s[c].scatter_(3, to, s[c].gather(3, source))
        source, to = (x[..., None].expand(n, b, hkv, t, DIM) for x in (source, to))
        for c in ("k", "v"):
            s[c].scatter_(3, to, s[c].gather(3, source))
        new_lens = s["lens"] + s["accepted"]
    return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"], "lens": new_lens}


def _sample(s):
    if own:
        from reef_b200 import kernels as K
        index, prob = K.sample_f32(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"index": index, "prob": prob}
    x = s["logits"]
    rows, n = x.shape
    greedy = s["temperature"] <= 0
    temperature = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    order = torch.argsort(x, dim=1, descending=True, stable=True)  # by value, then by index
    top = x.gather(1, order[:, :1]).double()
    w = torch.exp((x.double() - top) / temperature)  # 64 bits: a draw may lie next to a border
    rank = torch.arange(n, device=x.device)[None]
    ws = w.gather(1, order)
    keep = torch.ones_like(ws, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (k <= 0) | (rank < k)
    if s["top_p"] is not None:
        ws = ws * keep
        before = ws.cumsum(1) - ws
        p = s["top_p"].double()[:, None]
        keep &= (p >= 1) | (before < p * ws.sum(1, keepdim=True)) | (rank == 0)
    if s["min_p"] is not None:
        keep &= w.gather(1, order) >= s["min_p"].double()[:, None]
    keep &= ~greedy[:, None] | (rank == 0)
    w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    total = w.sum(1, keepdim=True)
    index = (w.cumsum(1) > s["u"].double()[:, None] * total).to(torch.uint8).argmax(1, keepdim=True)
    prob = w.gather(1, index) / total
    return {"index": index[:, 0].to(torch.int32), "prob": prob[:, 0].float()}


def _add_rms(s):
    if own:
        from reef_b200 import kernels as K
        h, codes, scale = K.add_rmsnorm_quant(s["x"], s["residual"], s["gain"], s["eps"])
    else:
        h = s["x"] + s["residual"]
        y = h * s["gain"] * (1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + s["eps"]))
        largest = y.abs().amax(1)
        scale = torch.where(largest > 0, largest / 127.0, torch.ones_like(largest))
        codes = torch.round(y / scale[:, None]).clamp(-127, 127)
    return {"h": h, "y": (codes.float() * scale[:, None]).bfloat16(), "scale": scale}


def _accept(s):
    if own:
        from reef_b200 import kernels as K
        path, accepted, following = K.tree_accept(s["tokens"], s["chosen"], parents=s["parents"])
        return {"path": path, "accepted": accepted, "next": following}
    parents, tokens, chosen = s["parents"].long(), s["tokens"], s["chosen"]
    b, t = tokens.shape
    i = torch.arange(t, device=tokens.device)
    hit = (chosen.gather(1, parents.clamp(min=0)) == tokens) & (parents >= 0)
    brothers = (parents[:, :, None] == parents[:, None, :]) & (i[None, :] < i[:, None])  # [b][i][j]: j an earlier child of i's parent
    hit &= ~(brothers & hit[:, None, :]).any(2)  # of equal children the first
    hit[:, 0] = True
    rooted = _ancestors(s["parents"])
    taken = (hit[:, None, :] | ~rooted).all(2) & rooted[:, :, 0]
    accepted = taken.sum(1)
    path = torch.where(taken, i[None], t).sort(1).values
    last = path.gather(1, accepted[:, None] - 1)
    path = torch.where(path < t, path, -1)
    return {"path": path.to(torch.int32), "accepted": accepted.to(torch.int32), "next": chosen.gather(1, last)[:, 0]}


def work(case):
    if case["op"] == "tree":
        keys = sum(n + d for n, d in zip(_lens(case), _draft_lens(case)))
        rows = sum(_draft_lens(case)) * case["heads_q"]
        seen = sum((n + (d + 1) / 2) * d for n, d in zip(_lens(case), _draft_lens(case))) * case["heads_q"]
        return {"bytes": keys * case["heads_kv"] * 2 * (DIM + 4) + rows * (DIM + 4 + 4 * DIM), "flops": 4.0 * DIM * seen}
    if case["op"] == "compact":
        moved = case["layers"] * case["batch"] * case["heads_kv"] * (case["drafts"] + 1) / 2
        return {"bytes": moved * 2 * 2 * (DIM + 4) + case["batch"] * (4 * case["drafts"] + 12), "flops": 0}
    if case["op"] == "sample":
        return {"bytes": 4 * case["rows"] * (case["n"] + 7), "flops": 4.0 * case["rows"] * case["n"]}
    if case["op"] == "add_rms":
        return {"bytes": case["rows"] * (13 * case["width"] + 4) + 4 * case["width"], "flops": 8.0 * case["rows"] * case["width"]}
    return {"bytes": case["batch"] * (16 * case["drafts"] + 8), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tree":
        out = s["out"].double()
        for b in range(case["batch"]):
            n, g = int(s["lens"][b]), case["heads_q"] // case["heads_kv"]
            parents = None if s["parents"] is None else s["parents"][b].tolist()
            d = case["drafts"] if s["draft_lens"] is None else int(s["draft_lens"][b])
            sees = torch.zeros((d, n + d), dtype=torch.bool)
            sees[:, :n] = True
            for i in range(d):
                j = i
                while j >= 0:
                    sees[i, n + j] = True
                    j = j - 1 if parents is None else parents[j]
            q = s["q8"][b, :d].double() * s["q_scale"][b, :d, :, None].double()
            k = s["k"][b, :, : n + d].double() * s["k_scale"][b, :, : n + d, None].double()
            v = s["v"][b, :, : n + d].double() * s["v_scale"][b, :, : n + d, None].double()
            sees = sees.cuda()
            for h in range(case["heads_q"]):
                x = torch.einsum("id,jd->ij", q[:, h], k[h // g]) * s["sm_scale"]
                out[b, :d, h] = torch.softmax(torch.where(sees, x, -math.inf), 1) @ v[h // g]
        return out
    if case["op"] == "compact":
        lens, path, accepted = s["lens"].tolist(), s["path"].tolist(), s["accepted"].tolist()
        got = {}
        for c in ("k_scale", "v_scale"):
            was = s[c].double()
            now = was.clone()
            for b in range(case["batch"]):
                for i in range(accepted[b]):
                    now[:, b, :, lens[b] + i] = was[:, b, :, lens[b] + path[b][i]]
            got[c] = now
        return {"k": None, "k_scale": got["k_scale"], "v": None, "v_scale": got["v_scale"], "lens": None}
    if case["op"] == "sample":
        x, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
        par = {k: None if s[k] is None else s[k].double().cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p")}
        prob = np.empty(case["rows"])
        for r in range(case["rows"]):
            if par["temperature"][r] <= 0:
                prob[r] = 1.0
                continue
            z = x[r] / par["temperature"][r]
            z = z - z.max()
            order = np.argsort(-x[r], kind="stable")
            if par["top_k"] is not None and par["top_k"][r] > 0:
                order = order[: int(par["top_k"][r])]
            if par["top_p"] is not None and par["top_p"][r] < 1:
                c = np.cumsum(np.exp(z[order]))
                order = order[: 1 + int(np.searchsorted(c[:-1], par["top_p"][r] * c[-1], side="left"))]
            if par["min_p"] is not None:
                order = order[np.exp(z[order]) >= par["min_p"][r]]
            kept = np.sort(order)
            c = np.cumsum(np.exp(z[kept]))
            at = int(np.searchsorted(c, u[r] * c[-1], side="right"))
            prob[r] = np.exp(z[kept[at]]) / c[-1]
        return {"index": None, "prob": torch.from_numpy(prob)}
    if case["op"] == "add_rms":
        h = s["x"].double() + s["residual"].double()
        y = h / torch.sqrt(torch.einsum("rw,rw->r", h, h)[:, None] / case["width"] + s["eps"]) * s["gain"].double()
        scale = y.abs().amax(1) / 127
        return {"h": h, "y": torch.round(y / scale[:, None]) * scale[:, None], "scale": scale}
    return None


if __name__ == "__main__":  # the cases, and some more of their ranges
    for one in listed() + [draw(random.Random(i)) for i in range(8)]:
        print(one, work(one))
