"""The calls whose speed is measured of what a decoder's layer has around its linears when it checks a tree of drafted tokens at once: the norms
before and after a block with its gate and residual scale, rotary positions of one or several axes, attention of the tree's tokens over a paged
cache, and the accepted path's move to its place in the cache.

Sequences of a batch lie one behind the other: `row_starts` says where the rows (drafted tokens) of each begin, `lengths` how many positions each has
with them, `pages` which page of the cache holds its positions.  `parents` says which row of its own sequence a row follows (-1: the last position
before the tree).  Row i of a sequence has place i behind what was accepted before, wherever it stands in the tree; the path that is then accepted
moves together (`accepted`: its rows, in their order).  What changes from call to call are the values, the trees, the pages and the caches'
contents; they come from the seed.  Sizes come from the case.  One pass is one dispatch of a program that was loaded before."""
import json
import math
import random

import torch

own = False  # set by who measures: the framework's operators, or their plain forms


def listed():
    return [
        # a decode step of eight conversations: behind a block its norm, the residual and the next block's norm, weights held less one
        dict(name="norm_8x1152", kind="norm", rows=8, N=1152, residual="bf16", post=True, gate="", offset=1.0, scale=1.0),
        # a prompt of ragged length, the block's result scaled by a gate for each token, an odd width
        dict(name="norm_777x2305_gated", kind="norm", rows=777, N=2305, residual="bf16", post=True, gate="row", offset=0.0, scale=1.0),
        # a batch of prompts with the residual held in 32 bits, a gate for each channel and a residual scale
        dict(name="norm_4096x4096_wide", kind="norm", rows=4096, N=4096, residual="f32", post=False, gate="channel", offset=0.0, scale=0.22),
        # the heads of a prompt's queries, each a row of its own
        dict(name="norm_heads_131072x128", kind="norm", rows=131072, N=128, residual="", post=False, gate="", offset=0.0, scale=1.0),
        # the drafted tokens of one conversation, four query heads and one key head of 256
        dict(name="rotary_16x256", kind="rotary", T=16, H=4, KVH=1, D=256, pairs=128, axes=1, interleaved=False, far=32768),
        # image patches far into a conversation, by height and width, a part of each head turned, neighbours paired
        dict(name="rotary_777x80_part", kind="rotary", T=777, H=16, KVH=16, D=80, pairs=16, axes=2, interleaved=True, far=1 << 20),
        # a video between text: time, height and width
        dict(name="rotary_8192x128_video", kind="rotary", T=8192, H=32, KVH=8, D=128, pairs=64, axes=3, interleaved=False, far=65536),
        # sixteen drafted tokens of one conversation
        dict(name="tree_bf16_1x16x1024", kind="tree", cache="bf16", S=1, new=16, context=1024, H=4, KVH=1, D=256, page=16, window=0, sinks=0, tail=0),
        # drafts of eight conversations in a layer with a sliding window, wide trees, pages of 24 positions
        dict(name="tree_bf16_8x200x4096_window", kind="tree", cache="bf16", S=8, new=200, context=4096, H=16, KVH=4, D=64, page=24, window=1024,
             sinks=4, tail=3),
        # drafts of sixteen long conversations on the quantised cache
        dict(name="tree_int8_16x64x8192", kind="tree", cache="int8", S=16, new=64, context=8192, H=32, KVH=8, D=128, page=64, window=0, sinks=0,
             tail=0),
        # what eight conversations accepted of their drafts
        dict(name="keep_bf16_8x16", kind="keep", cache="bf16", S=8, new=16, context=512, KVH=1, D=256, page=16, tail=0),
        # the same of 32 on the quantised cache, the accepted rows read back
        dict(name="keep_int8_32x64", kind="keep", cache="int8", S=32, new=64, context=1024, KVH=8, D=128, page=64, tail=0),
    ]


def _log(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "norm", "rotary", "rotary", "tree", "tree", "tree", "keep"])
        KVH, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 128, 256])
        if kind == "norm":
            N = rng.choice([D, _log(rng, 64, 16384), 8 * _log(rng, 64, 2048)])
            c = dict(kind=kind, rows=_log(rng, 1, 131072), N=N, residual=rng.choice(["", "bf16", "bf16", "f32"]), post=rng.random() < 0.5,
                     gate=rng.choice(["", "", "row", "channel", "element"]), offset=rng.choice([0.0, 1.0]), scale=rng.choice([1.0, 0.5, 0.22]))
        elif kind == "rotary":
            c = dict(kind=kind, T=_log(rng, 1, 32768), H=KVH * rng.choice([1, 2, 4, 8]), KVH=KVH, D=D, pairs=rng.choice([D // 2, D // 2, 8, 16]),
                     axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.4, far=_log(rng, 64, 1 << 20))
        else:
            context = _log(rng, 64, 32768)
            c = dict(kind=kind, cache=rng.choice(["bf16", "int8"]), S=_log(rng, 1, 64), new=min(context, rng.choice([1, _log(rng, 2, 512), _log(rng, 4, 128)])),
                     context=context, KVH=KVH, D=D, page=rng.choice([16, 16, 24, 32, 64, 128]), tail=rng.choice([0, 0, 1, 7]))
        if kind == "tree":
            c.update(H=KVH * rng.choice([1, 2, 4, 4, 8, 16]), window=0, sinks=0)
            if rng.random() < 0.4:
                c.update(window=_log(rng, 8, 4096), sinks=rng.choice([0, 1, 4, 16]))
        w = work(c)
        held = c["S"] * c["context"] * KVH * D if "S" in c else 0
        scores = c["S"] * c["new"] * c["context"] * c["H"] if kind == "tree" else 0
        if w["bytes"] <= 400e6 and w["flops"] <= 6e10 and held <= 1 << 28 and scores <= 1 << 29:
            return c


# ---- sizes ----------------------------------------------------------------------------------------------------------

def _sequences(case):
    """(drafted rows, positions with them, rows accepted) of each sequence, the same for every seed."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k not in ("name", "own")}, sort_keys=True))
    found = []
    for s in range(case["S"]):
        length = case["context"] if s == 0 else rng.randrange(1 + case["context"] // 3, case["context"] + 1)
        n = case["new"] if s == 0 or case["new"] <= 2 else rng.randrange(1 + case["new"] // 3, case["new"] + 1)
        n = min(n, length)
        found.append((n, length, min(n, rng.randrange(1, 9))))
    return found


def _rows(case):
    """Rows of the packed tensors: those of the sequences, and some behind the last one that nothing touches."""
    return sum(n for n, _, _ in _sequences(case)) + case["tail"]


def work(case):
    if case["kind"] == "norm":
        rows, N = case["rows"], case["N"]
        held = {"": 0, "bf16": 4, "f32": 8}[case["residual"]]  # read and written
        gate = {"": 0, "row": 2 * rows, "channel": 2 * N, "element": 2 * rows * N}[case["gate"]]
        return dict(bytes=rows * N * (4 + held) + 2 * N * (1 + case["post"]) + gate, flops=rows * N * (4 + 4 * case["post"] + 3 * bool(case["residual"])))
    if case["kind"] == "rotary":
        T, heads = case["T"], case["H"] + case["KVH"]
        return dict(bytes=4 * T * heads * case["D"] + 4 * T * case["axes"], flops=6 * T * heads * case["pairs"])
    KVH, D = case["KVH"], case["D"]
    stored = D + 4 if case["cache"] == "int8" else 2 * D  # bytes of a position's row in the cache, a key or a value
    index = 4 * (2 * case["S"] + 1)
    sequences = _sequences(case)
    if case["kind"] == "keep":
        kept = sum(k for _, _, k in sequences)
        back = 2 * kept * KVH * (stored + 2 * D) if case["cache"] == "int8" else 0
        return dict(bytes=2 * kept * KVH * 2 * stored + back + index + 4 * kept, flops=0)
    pairs = touched = 0
    for n, length, _ in sequences:
        first = length - n
        seen = min(first, case["window"] + min(first, case["sinks"])) if case["window"] else first
        pairs += n * (seen + 1)
        touched += seen + n
    rows = sum(n for n, _, _ in sequences)
    return dict(bytes=2 * rows * case["H"] * 2 * D + 2 * touched * KVH * stored + index + 4 * rows, flops=4 * pairs * case["H"] * D)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case, gen=gen)
    dict(norm=_prepare_norm, rotary=_prepare_rotary, tree=_prepare_cache, keep=_prepare_cache)[case["kind"]](case, s)
    del s["gen"]
    if own:
        _load(case, s)
    torch.cuda.synchronize()
    return s


def _normal(s, *shape):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=s["gen"]).to(torch.bfloat16)


def _uniform(s, *shape):
    return torch.rand(shape, dtype=torch.float32, device="cuda", generator=s["gen"])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_norm(case, s):
    rows, N = case["rows"], case["N"]
    # a few channels are much larger than the others, as a residual stream's are
    channels = torch.where(_uniform(s, N) < 0.01, 20.0, 1.0)
    s["input"] = (_normal(s, rows, N) * channels).to(torch.bfloat16)
    if case["residual"]:
        held = _normal(s, rows, N).float() * channels * 4.0
        s["residual"] = held.to(torch.bfloat16) if case["residual"] == "bf16" else held + 0.001 * _uniform(s, rows, N)
        s["sum"] = torch.empty_like(s["residual"])
    if case["gate"]:
        s["gate"] = torch.sigmoid(_normal(s, 1 if case["gate"] == "channel" else rows, 1 if case["gate"] == "row" else N).float() * 2).to(torch.bfloat16)
    for name in ("weight", "post_weight"):
        s[name] = (1.0 - case["offset"] + 0.3 * _normal(s, N).float()).to(torch.bfloat16)
    s["out"] = torch.empty_like(s["input"])


def _prepare_rotary(case, s):
    T, axes, pairs = case["T"], case["axes"], case["pairs"]
    s["query"], s["key"] = _normal(s, T, case["H"], case["D"]), _normal(s, T, case["KVH"], case["D"])
    s["query_out"], s["key_out"] = torch.empty_like(s["query"]), torch.empty_like(s["key"])
    s["frequencies"] = torch.tensor([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=torch.float32, device="cuda")
    s["axis_of"] = _ints([i * axes // pairs for i in range(pairs)])
    # some rows of text, which stand at one position on every axis, then pictures of 16 x 16 patches, one after another in time
    first = int(torch.randint(0, case["far"], (1,), device="cuda", generator=s["gen"]))
    at = torch.arange(T, device="cuda", dtype=torch.int64)
    patch = at - T // 8
    grid = [first + T // 8 + patch // 256, first + patch // 16 % 16, first + patch % 16][-axes:] if axes > 1 else [first + at]
    s["positions"] = torch.stack([torch.where(patch < 0, first + at, g) for g in grid]).to(torch.int32).contiguous()


def _prepare_cache(case, s):
    sequences, S, KVH, D, page = _sequences(case), case["S"], case["KVH"], case["D"], case["page"]
    starts = [0]
    for n, _, _ in sequences:
        starts.append(starts[-1] + n)
    s.update(row_starts=_ints(starts), lengths=_ints([length for _, length, _ in sequences]))
    # every sequence's pages are anywhere in the cache; what its table holds behind its last page is no page
    P = -(-case["context"] // page)
    NP = S * P + 3
    order = torch.randperm(NP, device="cuda", generator=s["gen"])[:S * P].to(torch.int32).reshape(S, P)
    used = torch.arange(P, device="cuda")[None, :] * page < s["lengths"][:, None]
    s["pages"] = torch.where(used, order, torch.full_like(order, -1)).contiguous()
    for name in ("key", "value"):
        if case["cache"] == "int8":
            s[name + "_cache"] = torch.randint(-127, 128, (NP, KVH, page, D), dtype=torch.int8, device="cuda", generator=s["gen"])
            s[name + "_scales"] = (_uniform(s, NP, KVH, page) + 0.5) * (1.0 / 73.3)
        else:
            s[name + "_cache"] = _normal(s, NP, KVH, page, D)
    rng = random.Random(int(torch.randint(0, 1 << 30, (1,), device="cuda", generator=s["gen"])))
    if case["kind"] == "tree":
        # a row's parent is any row a little before it: about half as deep as a chain would be at four rows, with up to a few tens at most
        parents = [max(-1, i - 1 - int(rng.expovariate(1.0) * (1 + i / 3))) for n, _, _ in sequences for i in range(n)]
        T = _rows(case)
        s["parents"] = _ints(parents + [0] * case["tail"])
        s["query"] = _normal(s, T, case["H"], D)
        s["out"] = _normal(s, T, case["H"], D)  # rows behind the last sequence keep what they hold
    else:
        kept = [sorted(rng.sample(range(n), k)) for n, _, k in sequences]
        most = max(len(k) for k in kept)
        s["accepted"] = _ints([k + [-1] * (most - len(k)) for k in kept])
        if case["cache"] == "int8":
            back = [0]
            for k in kept:
                back.append(back[-1] + len(k))
            s["read_starts"] = _ints(back)
            s["read_lengths"] = _ints([length - n + k for n, length, k in sequences])
            s["read_key"], s["read_value"] = _normal(s, back[-1], KVH, D), _normal(s, back[-1], KVH, D)


_the_device, _loaded = [], {}
_BINDINGS = {
    "norm": ["input", "residual", "gate", "weight", "post_weight", "sum", "out"],
    "rotary": ["query", "key", "positions", "query_out", "key_out"],
    "tree": ["query", "key_cache", "value_cache", "key_scales", "value_scales", "pages", "row_starts", "lengths", "parents", "out"],
    "keep": ["key_cache", "value_cache", "key_scales", "value_scales", "accepted", "pages", "row_starts", "lengths", "read_starts", "read_lengths",
             "read_key", "read_value"],
}


def _load(case, s):
    """The program of this case, serialised and loaded once, and the buffers of this state in the order of its bindings."""
    import numpy as np

    from torq_compiler_amd import Device, Executable, Program

    names = [name for name in _BINDINGS[case["kind"]] if name in s and (name != "post_weight" or case["post"])]
    if not _the_device:
        _the_device.append(Device(0))
    key = json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True)
    if key not in _loaded:
        types = {torch.bfloat16: np.uint16, torch.int8: np.int8, torch.int32: np.int32, torch.float32: np.float32}
        p = Program()
        v = {name: p.binding(i, tuple(s[name].shape), types[s[name].dtype]) for i, name in enumerate(names)}
        scales = dict(key_scales=v.get("key_scales"), value_scales=v.get("value_scales"))
        cache = [v[name] for name in ("key_cache", "value_cache", "pages") if name in v]
        if case["kind"] == "norm":
            p.norm(v["input"], v["weight"], eps=_EPS, weight_offset=case["offset"], residual=v.get("residual"), post_weight=v.get("post_weight"),
                   gate=v.get("gate"), residual_scale=case["scale"], residual_out=v.get("sum"), init=v["out"])
        elif case["kind"] == "rotary":
            p.rotary(v["query"], v["key"], v["positions"], s["frequencies"].cpu().numpy(), axes=s["axis_of"].cpu().numpy(),
                     interleaved=case["interleaved"], query_out=v["query_out"], key_out=v["key_out"])
        elif case["kind"] == "tree":
            p.tree_attention(v["query"], *cache, v["row_starts"], v["lengths"], v["parents"], scale=_scale(case), window=case["window"],
                             sinks=case["sinks"], init=v["out"], **scales)
        else:
            p.cache_keep(*cache, v["row_starts"], v["lengths"], v["accepted"], **scales)
            if case["cache"] == "int8":
                p.cache_read(*cache, v["read_starts"], v["read_lengths"], key=v["read_key"], value=v["read_value"], **scales)
        _loaded[key] = Executable(_the_device[0], p.serialize())
    buffers = [s[name] for name in names]
    s["executable"] = _loaded[key]
    s["pointers"] = [t.data_ptr() for t in buffers]
    s["sizes"] = [t.numel() * t.element_size() for t in buffers]


_EPS = 1e-6


def _scale(case):
    return 1.0 / math.sqrt(case["D"])


# ---- a pass ---------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        state["executable"].enqueue_device(state["pointers"], state["sizes"])
    else:
        dict(norm=_plain_norm, rotary=_plain_rotary, tree=_plain_tree, keep=_plain_keep)[case["kind"]](state)
    if case["kind"] == "norm":
        return [state["out"], state["sum"]] if case["residual"] else state["out"]
    if case["kind"] == "rotary":
        return [state["query_out"], state["key_out"]]
    if case["kind"] == "tree":
        return state["out"]
    if case["cache"] == "int8":
        return [state["read_key"], state["read_value"], state["key_scales"], state["value_scales"]]
    return [state["key_cache"], state["value_cache"]]


def _normed(x, weight, offset):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS) * (weight.float() + offset)


def _plain_norm(state):
    case = state["case"]
    x = state["input"].float()
    if case["post"]:
        x = _normed(x, state["post_weight"], case["offset"])
    if case["gate"]:
        x = x * state["gate"].float()
    if case["scale"] != 1.0:
        x = x * case["scale"]
    if case["residual"]:
        x = state["residual"].float() + x
        state["sum"].copy_(x)
    state["out"].copy_(_normed(x, state["weight"], case["offset"]))


def _plain_rotary(state):
    case = state["case"]
    n = case["pairs"]
    angle = state["positions"].double()[state["axis_of"].long()].T * state["frequencies"].double()  # [T, pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    for name in ("query", "key"):
        x, out = state[name].float(), state[name + "_out"]
        if case["interleaved"]:
            a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = x[..., :n], x[..., n:2 * n]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        out[..., :2 * n] = turned.to(torch.bfloat16)
        out[..., 2 * n:] = state[name][..., 2 * n:]


def _plain_tree(state):
    case = state["case"]
    S, H, KVH, D = case["S"], case["H"], case["KVH"], case["D"]
    starts, lengths = state["row_starts"], state["lengths"]
    n_max = max(n for n, _, _ in _sequences(case))
    n = starts[1:] - starts[:-1]
    row = torch.arange(n_max, device="cuda")
    at = (starts[:-1, None] + row).clamp_max(state["query"].shape[0] - 1)
    # the rows on each row's path, itself among them: parents, then twice as far each time
    parents = torch.where(row < n[:, None], state["parents"][at], torch.full_like(at, -1))
    path = ((parents[..., None] == row) | (row[:, None] == row)).float()
    for _ in range(max(1, (n_max - 1).bit_length())):
        path = torch.matmul(path, path).clamp_max_(1.0)
    depth = path.sum(dim=-1).to(torch.int32) - 1
    first = lengths - n
    pos = first[:, None] + depth  # [sequence, row]
    q = state["query"][at].float().reshape(S, n_max, KVH, H // KVH, D).permute(0, 2, 3, 1, 4).reshape(S, KVH, H // KVH * n_max, D)
    keys, values = _gathered(state, "key"), _gathered(state, "value")
    L = keys.shape[2]
    j = torch.arange(L, device="cuda")
    drafted = (j - first[:, None]).clamp(0, n_max - 1)  # [sequence, position]: the row that stands there, if one does
    where = torch.where(j < first[:, None], j.to(torch.int32), torch.gather(pos, 1, drafted))  # its position in the text
    seen = torch.gather(path, 2, drafted[:, None, :].expand(S, n_max, L)) > 0
    seen = torch.where(j < first[:, None, None], True, seen & (j < lengths[:, None, None]))
    if case["window"]:
        seen = seen & ((where[:, None] > pos[..., None] - case["window"]) | (where[:, None] < case["sinks"]))
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()).mul_(_scale(case)).reshape(S, KVH, H // KVH, n_max, L)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(most == -math.inf, torch.zeros_like(most), most)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    values = torch.where((j < lengths[:, None])[:, None, :, None], values, torch.zeros_like(values))
    o = torch.matmul(scores.reshape(S, KVH, H // KVH * n_max, L), values).reshape(S, KVH, H // KVH, n_max, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(S, n_max, H, D)
    rows = state["query"].shape[0] - case["tail"]
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    state["out"][:rows] = o[seq, (t - starts[seq]).long()].to(torch.bfloat16)


def _gathered(state, name):
    """Keys or values of every sequence, padded to the longest: [sequence, head, position, D] in 32 bits."""
    table = state["pages"].clamp_min(0).long()
    x = state[name + "_cache"][table].float()  # [sequence, page, head, slot, D]
    if state["case"]["cache"] == "int8":
        x *= state[name + "_scales"][table][..., None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_keep(state):
    case = state["case"]
    first = state["lengths"] - (state["row_starts"][1:] - state["row_starts"][:-1])
    seq, k = torch.nonzero(state["accepted"] >= 0, as_tuple=True)

    def place(position):
        return state["pages"][seq, (position // case["page"]).long()].long(), (position % case["page"]).long()

    source, to = place(first[seq] + state["accepted"][seq, k]), place(first[seq] + k.to(torch.int32))
    for name in ("key", "value"):
        for kind in ("_cache", "_scales"):
            if name + kind in state:
                state[name + kind][to[0], :, to[1]] = state[name + kind][source[0], :, source[1]]
        if case["cache"] == "int8":
            state["read_" + name].copy_(state[name + "_cache"][to[0], :, to[1]].float() * state[name + "_scales"][to[0], :, to[1]][..., None])


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        def norm(x, weight):
            return x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["N"] + _EPS) * (s[weight].double() + case["offset"])

        h = s["input"].double()
        if case["post"]:
            h = norm(h, "post_weight")
        h = h * s["gate"].double() * case["scale"] if case["gate"] else h * case["scale"]
        if not case["residual"]:
            return norm(h, "weight")
        h = s["residual"].double() + h
        return [norm(h, "weight"), h]
    if case["kind"] == "rotary":
        # pairs as complex numbers
        position = s["positions"].double()[s["axis_of"].long()]  # [pairs, T]
        turn = torch.polar(torch.ones_like(position), position * s["frequencies"].double()[:, None]).T[:, None]
        results = []
        for name in ("query", "key"):
            x = s[name].double()
            first, second = ((slice(0, 2 * case["pairs"], 2), slice(1, 2 * case["pairs"], 2)) if case["interleaved"] else
                             (slice(0, case["pairs"]), slice(case["pairs"], 2 * case["pairs"])))
            z = torch.complex(x[..., first], x[..., second]) * turn
            out = x.clone()
            out[..., first], out[..., second] = z.real, z.imag
            results.append(out)
        return results
    page, starts, lengths = case["page"], s["row_starts"].tolist(), s["lengths"].tolist()

    def places(i, positions):
        p = torch.tensor(positions, device="cuda")
        return s["pages"][i].long()[p // page], p % page

    def rows(i, name, positions):
        """What the cache holds at some positions of sequence i: [position, head, D]."""
        g, o = places(i, positions)
        x = s[name + "_cache"][g, :, o].double()
        return x * s[name + "_scales"][g, :, o].double()[..., None] if case["cache"] == "int8" else x

    if case["kind"] == "keep":
        moves = []
        for i, path in enumerate(s["accepted"].tolist()):
            first = lengths[i] - (starts[i + 1] - starts[i])
            path = [first + r for r in path if r >= 0]
            moves.append((path, list(range(first, first + len(path)))))
        result = []
        if case["cache"] == "int8":
            for name in ("key", "value"):
                result.append(torch.cat([rows(i, name, path) for i, (path, _) in enumerate(moves)]))
        for name in ("key_scales", "value_scales") if case["cache"] == "int8" else ("key_cache", "value_cache"):
            x = s[name].double()
            for i, (path, to) in enumerate(moves):
                (g, o), (tg, to) = places(i, path), places(i, to)
                x[tg, :, to] = s[name].double()[g, :, o]
            result.append(x)
        return result
    parents = s["parents"].tolist()
    out, G = s["out"].double(), case["H"] // case["KVH"]
    for i in range(case["S"]):
        n = starts[i + 1] - starts[i]
        first = lengths[i] - n
        hidden = torch.ones(n, lengths[i], dtype=torch.bool)
        depth = []
        for r in range(n):
            up = parents[starts[i] + r]
            depth.append(0 if up < 0 else depth[up] + 1)
            here = first + depth[r]
            low = max(0, here - case["window"] + 1) if case["window"] else 0
            hidden[r, min(low, first):first] = False
            hidden[r, :min(case["sinks"] if case["window"] else 0, first)] = False
            a = r
            while a >= 0:
                at = first + depth[a]
                if at >= low or at < case["sinks"]:
                    hidden[r, first + a] = False
                a = parents[starts[i] + a]
        hidden = hidden.cuda()
        q, keys, values = s["query"][starts[i]:starts[i + 1]].double(), *(rows(i, name, list(range(lengths[i]))) for name in ("key", "value"))
        for h in range(case["H"]):
            weights = (q[:, h] @ keys[:, h // G].T / math.sqrt(case["D"])).masked_fill(hidden, -math.inf)
            out[starts[i]:starts[i + 1], h] = torch.softmax(weights, dim=-1) @ values[:, h // G]
    return out
