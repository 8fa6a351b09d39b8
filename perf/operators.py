"""Operators of a decoding step over a key/value cache, with their plain forms and the cases that are measured.

tree     attention of the nodes of a tree of drafted tokens: every node sees its sequence's cached rows and, among the new
         rows, its ancestors and itself.  One node, or a chain of them, is an ordinary decoding step.
weights  the attention weight each cached row has received, added up over queries and the heads of a group: beside the
         attention of a decoding step, and for a whole prompt from the statistics its attention left.
evict    a cache cut down to a budget: the most recent rows and, of the others, those with the most weight, in order.
verify   the path of a drafted tree that the model's own choices confirm, and its keys and values appended to the caches
         of all layers.

Layouts: queries [batch, nodes, heads * headDim], caches [batch, capacity, kvHeads * headDim] with lengths[b] rows in use,
weights [batch, groups, capacity]; query head h reads key head h * kvHeads / heads and belongs to group h * groups / heads.
"""
import ctypes
import math
import random

import torch

own = False

# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # the GPT-small decoder, one sequence, one token: what a single step of generation costs, all latency
        dict(name="tree_one_token", op="tree", batch=1, heads=12, kv_heads=12, head_dim=64, nodes=1, capacity=1024, length=701, ragged=False),
        # a draft of 26 nodes over one long document, heads of the long-context decoder: a stream over 2 GB of cache
        dict(name="tree_long_document", op="tree", batch=1, heads=16, kv_heads=16, head_dim=128, nodes=26, capacity=131072, length=120011,
             ragged=False),
        # a serving batch of GPT-small sequences of all lengths, one of them empty, with full trees
        dict(name="tree_ragged_batch", op="tree", batch=32, heads=12, kv_heads=12, head_dim=64, nodes=64, capacity=4096, length=4032, ragged=True),
        # four query heads to a key head
        dict(name="tree_shared_heads", op="tree", batch=8, heads=32, kv_heads=8, head_dim=128, nodes=16, capacity=8192, length=8100, ragged=True),
        # one step of one GPT-small sequence that keeps account of the weight its cached rows receive
        dict(name="weights_one_token", op="weights", batch=1, heads=12, kv_heads=12, groups=12, head_dim=64, nodes=1, capacity=2048, length=1500,
             ragged=False),
        # the same for a batch of long sequences
        dict(name="weights_batch", op="weights", batch=16, heads=16, kv_heads=16, groups=16, head_dim=128, nodes=1, capacity=16384, length=16000,
             ragged=True),
        # the prompts of a GPT-small batch
        dict(name="weights_prompt", op="prompt", batch=8, heads=12, kv_heads=12, groups=12, head_dim=64, seq=1024, capacity=1024, ragged=False),
        # two long prompts of the long-context decoder, padded to one length
        dict(name="weights_long_prompt", op="prompt", batch=2, heads=16, kv_heads=16, groups=16, head_dim=128, seq=8192, capacity=8192, ragged=True),
        # one GPT-small sequence at the end of its cache, cut to half, every head keeping its own rows
        dict(name="evict_one", op="evict", batch=1, kv_heads=12, groups=12, head_dim=64, capacity=1024, length=1024, budget=512, recent=64,
             ragged=False),
        # a batch of long prompts cut to a quarter of the cache
        dict(name="evict_batch", op="evict", batch=8, kv_heads=16, groups=16, head_dim=128, capacity=16384, length=16384, budget=4096, recent=512,
             ragged=True),
        # a draft of 26 nodes of one GPT-small sequence: vocabulary of 50257, twelve layers
        dict(name="verify_one", op="verify", batch=1, nodes=26, vocab=50257, layers=12, kv_heads=12, head_dim=64, capacity=1024, length=700,
             ragged=False),
        # a serving batch with full trees, vocabulary of 32000
        dict(name="verify_batch", op="verify", batch=32, nodes=64, vocab=32000, layers=12, kv_heads=12, head_dim=64, capacity=512, length=440,
             ragged=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "prompt", "evict", "verify"])
    head_dim = rng.choice([64, 128, 64, 128, 32, 40, 80, 96, 100, 192, 256])
    batch, kv_heads = _spread(rng, 1, 32), _spread(rng, 1, 16)
    ragged = rng.random() < 0.6
    if op in ("tree", "weights"):
        nodes = _spread(rng, 1, 64)
        group = rng.choice([1, 1, 1, 2, 3, 4, 8]) if batch * nodes <= 512 else 1
        most = max(256, min(131072, (1 << 27) // (batch * kv_heads * head_dim)))
        capacity = max(nodes + 1, _spread(rng, 100, most))
        case = dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, nodes=nodes, capacity=capacity,
                    length=rng.randint(0, capacity - nodes) if rng.random() < 0.2 else capacity - nodes - rng.randint(0, (capacity - nodes) // 8),
                    ragged=ragged)
        if op == "weights":
            case["groups"] = rng.choice([1, kv_heads])
        return case
    if op == "prompt":
        group = rng.choice([1, 1, 2, 4])
        heads = kv_heads * group
        most = int(math.sqrt((1 << 31) / (batch * heads) * 64 / max(64, head_dim)))
        seq = _spread(rng, 1, max(2, min(8192, most)))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, groups=rng.choice([1, kv_heads]), head_dim=head_dim, seq=seq,
                    capacity=seq + rng.choice([0, 0, 37]), ragged=ragged)
    if op == "evict":
        most = max(512, min(65536, (1 << 28) // (batch * kv_heads * head_dim)))
        capacity = _spread(rng, 200, most)
        budget = rng.randint(1, capacity)
        return dict(op=op, batch=batch, kv_heads=kv_heads, groups=rng.choice([1, kv_heads]), head_dim=head_dim, capacity=capacity,
                    length=capacity - rng.randint(0, capacity // 8), budget=budget, recent=rng.randint(0, min(budget, 512)), ragged=ragged)
    nodes = _spread(rng, 1, 64)
    vocab = _spread(rng, 500, max(1000, min(260000, (1 << 26) // (batch * nodes))))
    layers = rng.randint(1, 24)
    kv_heads = rng.randint(1, 12)
    length = rng.randint(0, 300)
    return dict(op=op, batch=batch, nodes=nodes, vocab=vocab, layers=layers, kv_heads=kv_heads, head_dim=min(head_dim, 128),
                capacity=length + nodes + rng.randint(0, 64), length=length, ragged=ragged)


def _lengths(case):
    """Rows in use, sequence by sequence: `length` each, or spread over (0, length] with one empty sequence among three or more."""
    full = case["seq"] if case["op"] == "prompt" else case["length"]
    if not case["ragged"]:
        return [full] * case["batch"]
    spread = [math.ceil(full * (((i + 1) * 0.6180339887498949) % 1.0)) for i in range(case["batch"])]
    spread[0] = full
    if case["batch"] > 2 and case["op"] != "prompt":
        spread[1] = 0
    return spread


def _counts(case):
    """Nodes of each sequence's tree."""
    if not case["ragged"]:
        return [case["nodes"]] * case["batch"]
    return [max(1, case["nodes"] - (5 * i) % (case["nodes"] // 2 + 1)) for i in range(case["batch"])]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------


def _tree(case, seed):
    """Parents (a node's parent comes before it) and, as bits, the nodes each node sees: its ancestors and itself."""
    rng = random.Random(seed * 7919 + 17)
    parents, visible = [], []
    for _ in range(case["batch"]):
        p, see = [-1], [1]
        for j in range(1, case["nodes"]):
            p.append(rng.randrange(max(0, j - 6), j))
            see.append(see[p[j]] | 1 << j)
        parents.append(p)
        visible.append([v - (1 << 64) if v >= 1 << 63 else v for v in see])
    return torch.tensor(parents, dtype=torch.int32), torch.tensor(visible, dtype=torch.int64)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale)

    def zeros(*shape, dtype=torch.float32):
        return torch.zeros(*shape, device="cuda", dtype=dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32).cuda()

    op, b = case["op"], case["batch"]
    s = dict(case=case, op=op, lengths=ints(_lengths(case)))
    kv_dim, hd = case["kv_heads"] * case["head_dim"], case["head_dim"]
    if op in ("tree", "weights"):
        n, cap, dim = case["nodes"], case["capacity"], case["heads"] * hd
        parents, visible = _tree(case, seed)
        # logits of standard deviation 2: a few rows take most of the weight, as in trained heads
        s.update(q=normal(b, n, dim, scale=2.0), k_new=normal(b, n, kv_dim), v_new=normal(b, n, kv_dim), k=normal(b, cap, kv_dim),
                 v=normal(b, cap, kv_dim), counts=ints(_counts(case)), visible=visible.cuda(), scale=1.0 / math.sqrt(hd), out=zeros(b, n, dim),
                 m=zeros(b, case["heads"], n), l=zeros(b, case["heads"], n))
        if op == "weights":
            s.update(weights=normal(b, case["groups"], cap).square_(), weights_out=zeros(b, case["groups"], cap))
    elif op == "prompt":
        n, cap, heads = case["seq"], case["capacity"], case["heads"]
        s.update(q=normal(b, n, heads * hd, scale=2.0), k=normal(b, cap, kv_dim), scale=1.0 / math.sqrt(hd), weights_out=zeros(b, case["groups"], cap))
        # the statistics that the prompt's attention leaves
        scores = _prompt_scores(s)
        s["m"] = scores.amax(-1)
        s["l"] = scores.sub_(s["m"][..., None]).exp_().sum(-1)
    elif op == "evict":
        cap, budget = case["capacity"], case["budget"]
        s.update(k=normal(b, cap, kv_dim), v=normal(b, cap, kv_dim), weights=normal(b, case["groups"], cap).mul_(1.5).exp_(),
                 k_out=zeros(b, budget, kv_dim), v_out=zeros(b, budget, kv_dim), weights_out=zeros(b, case["groups"], budget),
                 kept=zeros(b, case["groups"], budget, dtype=torch.int32), lengths_out=zeros(b, dtype=torch.int32))
    else:
        n, vocab, cap, layers = case["nodes"], case["vocab"], case["capacity"], case["layers"]
        parents, visible = _tree(case, seed)
        parents = parents.cuda()
        tokens = torch.randint(0, vocab, (b, n), generator=gen, device="cuda")
        logits = normal(b, n, vocab, scale=3.0)
        # the model agrees with about half of the drafted tokens
        agree = torch.rand(b, n, generator=gen, device="cuda") < 0.5
        agree[:, 0] = False
        row = torch.arange(b, device="cuda")[:, None].expand(b, n)
        logits.index_put_((row[agree], parents.long()[agree], tokens[agree]), torch.tensor(25.0, device="cuda"))
        s.update(logits=logits, tokens=tokens.float(), parents=parents, visible=visible.cuda(), counts=ints(_counts(case)),
                 k_new=normal(layers, b, n, kv_dim), v_new=normal(layers, b, n, kv_dim), k=normal(layers, b, cap, kv_dim),
                 v=normal(layers, b, cap, kv_dim), path=zeros(b, n, dtype=torch.int32), path_counts=zeros(b, dtype=torch.int32), next=zeros(b),
                 lengths_out=zeros(b, dtype=torch.int32))
        for name in ("k", "v", "k_new", "v_new"):   # a layer's tensor at a time, as a model holds them
            s["each_" + name] = (ctypes.c_void_p * layers)(*[t.data_ptr() for t in s[name]])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------


def _bits(visible, n):
    return (visible[..., None] >> torch.arange(n, device=visible.device)) & 1 != 0


def _prompt_scores(s):
    """Scaled scores of a causal prompt, [batch, heads, seq, seq], minus infinity where a query does not see the key."""
    c = s["case"]
    b, n, kv, hd = c["batch"], c["seq"], c["kv_heads"], c["head_dim"]
    q = s["q"].view(b, n, kv, -1, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hd)
    k = s["k"][:, :n].view(b, n, kv, hd).permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(q, k).mul_(s["scale"]).view(b, c["heads"], n, n)
    at = torch.arange(n, device=q.device)
    return scores.masked_fill_(at[None, :] > at[:, None], -math.inf)


def _attention(s):
    """Probabilities over the cached and over the new rows, the output and its statistics."""
    c = s["case"]
    b, n, cap, heads, kv, hd = c["batch"], c["nodes"], c["capacity"], c["heads"], c["kv_heads"], c["head_dim"]
    q = s["q"].view(b, n, kv, -1, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hd)
    live = torch.arange(n, device=q.device)[None] < s["counts"][:, None]

    def split(x):
        return x.view(b, -1, kv, hd).permute(0, 2, 1, 3).contiguous()

    cached = torch.matmul(q, split(s["k"]).transpose(2, 3)).view(b, heads, n, cap) * s["scale"]
    fresh = torch.matmul(q, split(s["k_new"]).transpose(2, 3)).view(b, heads, n, n) * s["scale"]
    used = torch.arange(cap, device=q.device)[None] < s["lengths"][:, None]
    cached = cached.masked_fill(~used[:, None, None, :], -math.inf)
    fresh = fresh.masked_fill(~(_bits(s["visible"], n) & live[:, None, :])[:, None], -math.inf)
    m = torch.maximum(cached.amax(-1), fresh.amax(-1))
    about = torch.where(m == -math.inf, 0.0, m)[..., None]
    p_cached, p_fresh = torch.exp(cached - about), torch.exp(fresh - about)
    l = p_cached.sum(-1) + p_fresh.sum(-1)
    over = torch.where(l > 0, 1.0 / l, 0.0)[..., None]
    p_cached, p_fresh = p_cached * over, p_fresh * over
    out = (torch.matmul(p_cached.view(b, kv, -1, cap), split(s["v"])) + torch.matmul(p_fresh.view(b, kv, -1, n), split(s["v_new"])))
    out = out.view(b, heads, n, hd).permute(0, 2, 1, 3).reshape(b, n, -1)
    out = torch.where(live[:, :, None], out, s["out"])
    m, l = torch.where(live[:, None], m, s["m"]), torch.where(live[:, None], l, s["l"])
    return live, p_cached, p_fresh, out, m, l


def _plain_weights(s):
    c = s["case"]
    b, n, cap, groups = c["batch"], c["nodes"], c["capacity"], c["groups"]
    live, p_cached, p_fresh, out, m, l = _attention(s)

    def gathered(p):   # over the nodes in use, then over the heads of a group
        return (p * live[:, None, :, None]).sum(2).view(b, groups, -1, p.shape[-1]).sum(2)

    cached, fresh = gathered(p_cached), gathered(p_fresh)
    at = torch.arange(cap, device=cached.device)[None]
    length = s["lengths"][:, None]
    rank = (at - length).clamp(0, n - 1)[:, None].expand(b, groups, cap)
    new = (at >= length) & (at < length + s["counts"][:, None])
    total = torch.where((at < length)[:, None], s["weights"] + cached, s["weights_out"])
    return [out, m, l, torch.where(new[:, None], fresh.gather(2, rank), total)]


def _plain_prompt(s):
    c = s["case"]
    b, n, groups = c["batch"], c["seq"], c["groups"]
    p = torch.exp(_prompt_scores(s) - s["m"][..., None]) / s["l"][..., None]
    live = torch.arange(n, device=p.device)[None] < s["lengths"][:, None]
    total = (p * live[:, None, :, None]).sum(2).view(b, groups, -1, n).sum(2)
    return torch.cat([total, s["weights_out"][..., n:]], 2)


def _plain_evict(s):
    c = s["case"]
    b, cap, groups, budget = c["batch"], c["capacity"], c["groups"], c["budget"]
    length = s["lengths"][:, None, None]
    at = torch.arange(cap, device=length.device)
    kind = (at < length).int() + ((at < length) & (at >= length - c["recent"])).int()   # 2: recent, 1: by weight, 0: not in use
    kind = kind.expand(b, groups, cap)
    weight = torch.where(torch.isnan(s["weights"]), -math.inf, s["weights"]) + 0.0
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices
    order = order.gather(2, torch.sort(kind.gather(2, order), dim=-1, descending=True, stable=True).indices)[..., :budget]
    left = length.clamp(max=budget)
    valid = torch.arange(budget, device=at.device) < left
    kept = torch.sort(torch.where(valid, order, cap), dim=-1).values
    kept = torch.where(valid, kept, 0)

    def rows(x, old):
        x = x.view(b, cap, groups, -1)
        index = kept.permute(0, 2, 1)[..., None].expand(b, budget, groups, x.shape[-1])
        return torch.where(valid.permute(0, 2, 1)[..., None], x.gather(1, index), old.view(b, budget, groups, -1)).view(b, budget, -1)

    weights = torch.where(valid, s["weights"].gather(2, kept), s["weights_out"])
    return [rows(s["k"], s["k_out"]), rows(s["v"], s["v_out"]), weights, torch.where(valid, kept.int(), s["kept"]), left[:, 0, 0].int()]


def _plain_verify(s):
    c = s["case"]
    b, n, vocab, layers = c["batch"], c["nodes"], c["vocab"], c["layers"]
    at = torch.arange(n, device=s["tokens"].device)
    top = s["logits"].amax(-1, keepdim=True)
    choice = torch.where(s["logits"] == top, torch.arange(vocab, device=at.device), vocab).amin(-1)
    parents, tokens = s["parents"].long(), s["tokens"].round().long()
    live = at[None] < s["counts"][:, None]
    twin = (parents[:, :, None] == parents[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :]) & (at[None, :] < at[:, None])
    fits = (tokens == choice.gather(1, parents.clamp(min=0))) & ~(twin & live[:, None, :]).any(-1)
    fits = (fits | (at == 0)) & live
    on_path = ~(_bits(s["visible"], n) & ~fits[:, None, :]).any(-1)
    count = on_path.sum(-1)
    path = torch.sort(torch.where(on_path, at, n), dim=-1).values
    valid = at[None] < count[:, None]
    chosen = choice.gather(1, path.gather(1, (count - 1).clamp(min=0)[:, None]).clamp(max=n - 1))[:, 0]
    # a path longer than the rest of the cache is not appended; the cases leave room for every node
    row = path.clamp(max=n - 1)[None, :, :, None].expand(layers, b, n, s["k"].shape[-1])
    target = (s["lengths"][:, None] + at).long()[None, :, :, None].expand_as(row)
    keep = valid[None, :, :, None]
    for cache, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        cache.scatter_(2, target, torch.where(keep, new.gather(2, row), cache.gather(2, target)))
    return [torch.where(valid, path, -1).int(), count.int(), chosen.float(), s["lengths"] + count.int(), s["k"], s["v"]]


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------


def _ours(s):
    from blackforge_amd import capi

    c, call = s["case"], capi.call

    def p(name):
        return s[name].data_ptr()

    if s["op"] == "tree":
        call("bf_hip_attention_tree", p("q"), p("k_new"), p("v_new"), p("k"), p("v"), p("lengths"), p("counts"), p("visible"), p("out"), p("m"),
             p("l"), c["batch"], c["heads"], c["kv_heads"], c["nodes"], c["capacity"], c["head_dim"], s["scale"], None)
        return [s["out"], s["m"], s["l"]]
    if s["op"] == "weights":
        call("bf_hip_attention_tree_weights", p("q"), p("k_new"), p("v_new"), p("k"), p("v"), p("lengths"), p("counts"), p("visible"), p("out"),
             p("m"), p("l"), p("weights"), p("weights_out"), c["batch"], c["heads"], c["kv_heads"], c["groups"], c["nodes"], c["capacity"],
             c["head_dim"], s["scale"], None)
        return [s["out"], s["m"], s["l"], s["weights_out"]]
    if s["op"] == "prompt":
        call("bf_hip_attention_key_weights", p("q"), p("k"), p("m"), p("l"), p("lengths"), None, p("weights_out"), c["batch"], c["heads"],
             c["kv_heads"], c["groups"], c["seq"], c["seq"], c["capacity"], c["head_dim"], s["scale"], 0, c["capacity"], None)
        return s["weights_out"]
    if s["op"] == "evict":
        call("bf_hip_kv_evict", p("k"), p("v"), p("weights"), p("lengths"), p("k_out"), p("v_out"), p("weights_out"), p("lengths_out"), p("kept"),
             c["batch"], c["kv_heads"], c["groups"], c["head_dim"], c["capacity"], c["budget"], c["budget"], c["recent"], None)
        return [s["k_out"], s["v_out"], s["weights_out"], s["kept"], s["lengths_out"]]
    call("bf_hip_tree_accept", p("logits"), p("tokens"), p("parents"), p("counts"), p("path"), p("path_counts"), p("next"), c["batch"], c["nodes"],
         c["vocab"], None)
    call("bf_hip_kv_commit", s["each_k"], s["each_v"], s["each_k_new"], s["each_v_new"], None, c["layers"], p("path"), p("path_counts"),
         p("lengths"), p("lengths_out"), c["batch"], c["kv_heads"], 1, c["nodes"], c["capacity"], c["head_dim"], None)
    return [s["path"], s["path_counts"], s["next"], s["lengths_out"], s["k"], s["v"]]


def run(state):
    if own:
        return _ours(state)
    if state["op"] == "tree":
        return list(_attention(state)[3:])
    if state["op"] == "weights":
        return _plain_weights(state)
    if state["op"] == "prompt":
        return _plain_prompt(state)
    if state["op"] == "evict":
        return _plain_evict(state)
    return _plain_verify(state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    b, hd, kv_dim = case["batch"], case["head_dim"], case["kv_heads"] * case["head_dim"]
    lengths = _lengths(case)
    if case["op"] in ("tree", "weights"):
        counts, heads = _counts(case), case["heads"]
        read = 4 * (2 * kv_dim * (sum(lengths) + sum(counts)) + 2 * heads * hd * sum(counts) + 2 * heads * sum(counts))
        if case["op"] == "weights":
            read += 8 * case["groups"] * sum(lengths)
        return {"bytes": read, "flops": sum(4 * hd * heads * n * (length + (n + 1) // 2) for n, length in zip(counts, lengths))}
    if case["op"] == "prompt":
        n, heads = case["seq"], case["heads"]
        return {"bytes": 4 * (sum(lengths) * (heads * hd + kv_dim + 2 * heads) + b * case["groups"] * n),
                "flops": sum(2 * hd * heads * (x * (x + 1) // 2) for x in lengths)}
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lengths)
        return {"bytes": 4 * (4 * kv_dim * kept + case["groups"] * (sum(lengths) + 2 * kept)), "flops": case["groups"] * sum(lengths)}
    nodes = sum(_counts(case))
    return {"bytes": 4 * (nodes * case["vocab"] + 4 * case["layers"] * b * 2 * kv_dim), "flops": nodes * case["vocab"]}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] in ("evict", "verify"):   # copies and indices: nothing is computed
        return None
    s = prepare(case, seed)
    heads, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    share = heads // kv
    if case["op"] == "prompt":
        n, groups = case["seq"], case["groups"]
        total = torch.zeros_like(s["weights_out"], dtype=torch.float64)
        future = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for i, count in enumerate(_lengths(case)):
            for h in range(heads):
                q = s["q"][i, :count, h * hd:(h + 1) * hd].double()
                k = s["k"][i, :n, h // share * hd:(h // share + 1) * hd].double()
                score = (q @ k.t()) * s["scale"] - s["m"][i, h, :count, None].double()
                score[future[:count]] = -math.inf
                total[i, h * groups // heads, :n] += (torch.exp(score) / s["l"][i, h, :count, None].double()).sum(0)
        return total
    out, m, l = (s[name].double() for name in ("out", "m", "l"))
    if case["op"] == "weights":
        weights = s["weights_out"].double()
    for i, (length, count) in enumerate(zip(_lengths(case), _counts(case))):
        masks = s["visible"][i].tolist()
        sees = torch.tensor([[j < length or masks[r] >> (j - length) & 1 == 1 for j in range(length, length + count)] for r in range(count)]).cuda()
        sees = torch.cat([torch.ones(count, length, dtype=torch.bool, device="cuda"), sees], 1)
        for g in range(kv):
            k = torch.cat([s["k"][i, :length, g * hd:(g + 1) * hd], s["k_new"][i, :count, g * hd:(g + 1) * hd]]).double()
            v = torch.cat([s["v"][i, :length, g * hd:(g + 1) * hd], s["v_new"][i, :count, g * hd:(g + 1) * hd]]).double()
            for h in range(g * share, (g + 1) * share):
                score = s["q"][i, :count, h * hd:(h + 1) * hd].double() @ k.t() * s["scale"]
                score[~sees] = -math.inf
                top = score.max(1).values
                e = torch.exp(score - top[:, None])
                total = e.sum(1)
                m[i, h, :count], l[i, h, :count] = top, total
                out[i, :count, h * hd:(h + 1) * hd] = e @ v / total[:, None]
                if case["op"] == "weights":
                    got, at = (e / total[:, None]).sum(0), h * case["groups"] // heads
                    if h % (heads // case["groups"]) == 0:
                        weights[i, at, :length] = s["weights"][i, at, :length]
                        weights[i, at, length:length + count] = 0
                    weights[i, at, :length + count] += got
    return [out, m, l, weights] if case["op"] == "weights" else [out, m, l]
