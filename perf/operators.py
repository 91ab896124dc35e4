"""The calls whose speed is measured of the operators around a decoder's cache: writing new keys and values into a paged
cache (as bf16, or quantised to int8), reading a cache back, attention over the prompts of a batch, and attention of a
chunk of new tokens over the paged cache.

Sequences of a batch lie one behind the other: `row_starts` says where the rows (tokens) of each begin, `lengths` how many
positions each has with the new ones, `pages` which page of the cache holds its positions.  What changes from call to call
are the values, the pages and the caches' contents; they come from the seed.  Lengths come from the case.  One pass is one
dispatch of a program that was loaded before."""
import json
import math
import random

import torch

own = False  # set by who measures: the framework's operators, or their plain forms


def listed():
    return [
        # a decode step of eight conversations: one new token each, one key / value head of 256
        dict(name="write_bf16_8x1", kind="write", cache="bf16", S=8, new=1, context=1024, KVH=1, D=256, page=16, tail=0),
        # a batch of prompts goes into the cache
        dict(name="write_bf16_8192", kind="write", cache="bf16", S=5, new=3500, context=4096, KVH=8, D=128, page=16, tail=13),
        # one more token for each of 32 conversations, quantised; all of them read back (to move them to another server)
        dict(name="append_read_int8_32x1024", kind="append_read", cache="int8", S=32, new=1, context=1024, KVH=1, D=256, page=16, tail=0),
        # long documents read back from the quantised cache
        dict(name="read_int8_4x8192", kind="read", cache="int8", S=4, new=8192, context=8192, KVH=8, D=128, page=64, tail=0),
        # a few short prompts with a sliding window, four query heads over one key / value head
        dict(name="prompt_4x128_window", kind="attention", S=4, new=128, H=4, KVH=1, D=256, window=64, sinks=0, tail=0),
        # a batch of ragged prompts, every earlier token visible
        dict(name="prompt_6x2048", kind="attention", S=6, new=2048, H=4, KVH=1, D=256, window=0, sinks=0, tail=5),
        # one long document with a sliding window and its first tokens
        dict(name="prompt_1x8192_sinks", kind="attention", S=1, new=8192, H=32, KVH=8, D=128, window=1024, sinks=4, tail=0),
        # the next token of one conversation
        dict(name="decode_bf16_1x1024", kind="paged", cache="bf16", S=1, new=1, context=1024, H=4, KVH=1, D=256, page=16, window=0, sinks=0,
             tail=0),
        # the next token of 32 conversations in a layer with a sliding window, on the quantised cache
        dict(name="decode_int8_32x1024_window", kind="paged", cache="int8", S=32, new=1, context=1024, H=4, KVH=1, D=256, page=16, window=512,
             sinks=4, tail=0),
        # the next token of 16 long conversations on the quantised cache
        dict(name="decode_int8_16x32768", kind="paged", cache="int8", S=16, new=1, context=32768, H=32, KVH=8, D=128, page=64, window=0,
             sinks=0, tail=0),
        # prompts read in chunks of 512, over what the cache holds of them
        dict(name="chunk_bf16_4x512x8192", kind="paged", cache="bf16", S=4, new=512, context=8192, H=32, KVH=8, D=128, page=64, window=0,
             sinks=0, tail=0),
        # conversations and one prompt's chunk in one batch, heads of 64, pages of 24 positions
        dict(name="mixed_int8_24x777x4096", kind="paged", cache="int8", S=24, new=777, mixed=True, context=4096, H=16, KVH=4, D=64, page=24,
             window=2048, sinks=16, tail=3),
    ]


def _log(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["write", "append_read", "read", "attention", "attention", "paged", "paged", "paged"])
    while True:
        KVH = rng.choice([1, 2, 4, 8])
        D = rng.choice([64, 80, 96, 128, 128, 256])
        c = dict(kind=kind, S=_log(rng, 1, 64), KVH=KVH, D=D, tail=rng.choice([0, 0, 1, 7]))
        if kind == "attention":
            c.update(H=KVH * rng.choice([1, 2, 4, 4, 8]), new=_log(rng, 1, 8192), window=0, sinks=0)
        else:
            c.update(cache="int8" if kind == "append_read" else rng.choice(["bf16", "int8"]) if kind in ("read", "paged") else "bf16",
                     page=rng.choice([16, 16, 24, 32, 64, 128]), context=_log(rng, 16, 32768))
            c["new"] = c["context"] if kind == "read" else min(c["context"], rng.choice([1, 1, _log(rng, 1, 8), _log(rng, 1, 4096)]))
        if kind == "paged":
            c.update(H=KVH * rng.choice([1, 2, 4, 4, 8, 16]), window=0, sinks=0, mixed=rng.random() < 0.2)
        if kind in ("attention", "paged") and rng.random() < 0.5:
            c.update(window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 16]))
        w = work(c)
        scores = max((n for n, _ in _sequences(c)), default=0) * _longest(c) * c["S"] * c.get("H", 0)
        if w["bytes"] <= 400e6 and w["flops"] <= 1.25e11 and scores <= 1 << 31 and c["S"] * _longest(c) * KVH * D <= 1 << 29:
            return c


# ---- lengths --------------------------------------------------------------------------------------------------------

def _sequences(case):
    """(new rows, positions with them) of each sequence, the same for every seed."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k not in ("name", "own")}, sort_keys=True))
    found = []
    for s in range(case["S"]):
        n = case["new"] if s == 0 or case["new"] <= 2 else rng.randrange(1 + case["new"] // 3, case["new"] + 1)
        if case.get("mixed") and s > 0:
            n = 1  # a conversation beside the prompt
        if case["kind"] == "attention":
            found.append((n, n))
            continue
        length = case["context"] if s == 0 else rng.randrange(1 + case["context"] // 3, case["context"] + 1)
        found.append((min(n, length) if case["kind"] != "read" else length, length))
    return found


def _longest(case):
    return max(length for _, length in _sequences(case))


def _rows(case):
    """Rows of the packed tensors: those of the sequences, and some behind the last one that nothing touches."""
    return sum(n for n, _ in _sequences(case)) + case["tail"]


def _table_pages(case):
    return -(-case.get("context", 1) // case.get("page", 1))


def _spans(case):
    """(visible pairs of a row and a position, positions that some row sees) over the batch."""
    pairs = touched = 0
    window, sinks = case["window"], case["sinks"]
    for n, length in _sequences(case):
        first = length - n
        if not window:
            pairs += n * first + n * (n + 1) // 2
            touched += length
            continue
        for p in range(first, length):
            low = max(0, p + 1 - window)
            pairs += p + 1 - low + min(sinks, low)
        low = max(0, first + 1 - window)
        touched += length - low + min(sinks, low)
    return pairs, touched


def work(case):
    KVH, D = case["KVH"], case["D"]
    stored = D + 4 if case.get("cache") == "int8" else 2 * D  # bytes of a position's row in the cache, a key or a value
    rows = sum(n for n, _ in _sequences(case))
    held = sum(length for _, length in _sequences(case))
    index = 4 * (2 * case["S"] + 1)
    if case["kind"] == "write":
        return dict(bytes=2 * rows * KVH * (2 * D + stored) + index, flops=0)
    if case["kind"] == "read":
        return dict(bytes=2 * rows * KVH * (2 * D + stored) + index, flops=0)
    if case["kind"] == "append_read":
        return dict(bytes=2 * rows * KVH * (2 * D + stored) + 2 * held * KVH * (2 * D + stored) + index, flops=0)
    pairs, touched = _spans(case)
    if case["kind"] == "attention":
        stored = 2 * D
    return dict(bytes=2 * rows * case["H"] * 2 * D + 2 * touched * KVH * stored + index, flops=4 * pairs * case["H"] * D)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sequences, S, KVH, D, T = _sequences(case), case["S"], case["KVH"], case["D"], _rows(case)

    def normal(*shape):
        return torch.randn(shape, dtype=torch.float32, device="cuda", generator=gen).to(torch.bfloat16)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    starts = [0]
    for n, _ in sequences:
        starts.append(starts[-1] + n)
    s = dict(case=case, row_starts=ints(starts), lengths=ints([length for _, length in sequences]))
    if case["kind"] == "append_read":  # the rows that are read: all positions of each sequence
        held = [0]
        for _, length in sequences:
            held.append(held[-1] + length)
        s["read_starts"] = ints(held)
    if case["kind"] != "attention":
        # every sequence's pages are anywhere in the cache; what its table holds behind its last page is no page
        page, P = case["page"], _table_pages(case)
        NP = S * P + 3
        order = torch.randperm(NP, device="cuda", generator=gen)[:S * P].to(torch.int32).reshape(S, P)
        used = torch.arange(P, device="cuda")[None, :] * page < s["lengths"][:, None]
        s["pages"] = torch.where(used, order, torch.full_like(order, -1)).contiguous()
        for name in ("key", "value"):
            if case["cache"] == "int8":
                s[name + "_cache"] = torch.randint(-127, 128, (NP, KVH, page, D), dtype=torch.int8, device="cuda", generator=gen)
                s[name + "_scales"] = (torch.rand(NP, KVH, page, device="cuda", generator=gen) + 0.5) * (1.0 / 73.3)
            else:
                s[name + "_cache"] = normal(NP, KVH, page, D)
    if case["kind"] in ("write", "append_read", "attention"):
        # single rows are larger or smaller than others, as a decoder's are
        grow = torch.exp(0.5 * torch.randn(T, 1, 1, device="cuda", generator=gen)) if case["kind"] != "attention" else 1.0
        s["key"], s["value"] = ((normal(T, KVH, D) * grow).to(torch.bfloat16) for _ in range(2))
    if case["kind"] in ("attention", "paged"):
        s["query"] = normal(T, case["H"], D)
        s["out"] = normal(T, case["H"], D)  # rows behind the last sequence keep what they hold
    if case["kind"] in ("read", "append_read"):
        R = T if case["kind"] == "read" else sum(length for _, length in sequences)
        s["read_key"], s["read_value"] = normal(R, KVH, D), normal(R, KVH, D)
    if own:
        _load(case, s)
    torch.cuda.synchronize()
    return s


_the_device, _loaded = [], {}
_BINDINGS = {
    "write": ["key", "value", "key_cache", "value_cache", "pages", "row_starts", "lengths"],
    "read": ["key_cache", "value_cache", "pages", "row_starts", "lengths", "read_key", "read_value"],
    "append_read": ["key", "value", "key_cache", "value_cache", "pages", "row_starts", "lengths", "read_starts", "read_key", "read_value"],
    "attention": ["query", "key", "value", "row_starts", "out"],
    "paged": ["query", "key_cache", "value_cache", "pages", "row_starts", "lengths", "out"],
}


def _load(case, s):
    """The program of this case, serialised and loaded once, and the buffers of this state in the order of its bindings."""
    import numpy as np

    from torq_compiler_amd import Device, Executable, Program

    names = _BINDINGS[case["kind"]] + (["key_scales", "value_scales"] if case.get("cache") == "int8" else [])
    if not _the_device:
        _the_device.append(Device(0))
    key = json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True)
    if key not in _loaded:
        types = {torch.bfloat16: np.uint16, torch.int8: np.int8, torch.int32: np.int32, torch.float32: np.float32}
        p = Program()
        v = {name: p.binding(i, tuple(s[name].shape), types[s[name].dtype]) for i, name in enumerate(names)}
        scales = dict(key_scales=v.get("key_scales"), value_scales=v.get("value_scales"))
        cache = [v[name] for name in ("key_cache", "value_cache", "pages") if name in v]
        if case["kind"] in ("write", "append_read"):
            p.cache_write(v["key"], v["value"], *cache, v["row_starts"], v["lengths"], **scales)
        if case["kind"] in ("read", "append_read"):
            p.cache_read(*cache, v.get("read_starts", v["row_starts"]), v["lengths"], key=v["read_key"], value=v["read_value"], **scales)
        see = dict(scale=_scale(case), window=case["window"], sinks=case["sinks"], init=v["out"]) if "H" in case else {}
        if case["kind"] == "attention":
            p.attention(v["query"], v["key"], v["value"], v["row_starts"], **see)
        if case["kind"] == "paged":
            p.paged_attention(v["query"], *cache, v["row_starts"], v["lengths"], **see, **scales)
        _loaded[key] = Executable(_the_device[0], p.serialize())
    buffers = [s[name] for name in names]
    s["executable"] = _loaded[key]
    s["pointers"] = [t.data_ptr() for t in buffers]
    s["sizes"] = [t.numel() * t.element_size() for t in buffers]


def _scale(case):
    return 1.0 / math.sqrt(case["D"])


# ---- a pass ---------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        state["executable"].enqueue_device(state["pointers"], state["sizes"])
    elif case["kind"] == "write":
        _plain_write(state)
    elif case["kind"] == "append_read":
        _plain_write(state)
        _plain_read(state, state["read_starts"])
    elif case["kind"] == "read":
        _plain_read(state, state["row_starts"])
    else:
        _plain_attention(state)
    if case["kind"] == "write":
        return [state["key_cache"], state["value_cache"]]
    if case["kind"] == "append_read":
        return [state["read_key"], state["read_value"], state["key_scales"], state["value_scales"]]
    if case["kind"] == "read":
        return [state["read_key"], state["read_value"]]
    return state["out"]


def _places(state, starts, rows):
    """Sequence and position of each of the first `rows` rows."""
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    return seq, (state["lengths"] - starts[1:])[seq] + at


def _plain_write(state):
    case = state["case"]
    rows = state["key"].shape[0] - case["tail"]
    seq, pos = _places(state, state["row_starts"], rows)
    page = state["pages"][seq, (pos // case["page"]).long()].long()
    slot = (pos % case["page"]).long()
    for name in ("key", "value"):
        x = state[name][:rows]
        if case["cache"] == "int8":
            x = x.float()
            most = x.abs().amax(dim=-1).clamp_min(2.0 ** -100)
            state[name + "_scales"][page, :, slot] = most / 127.0
            x = torch.round(x * (127.0 / most)[..., None]).to(torch.int8)
        state[name + "_cache"][page, :, slot] = x


def _plain_read(state, starts):
    case = state["case"]
    rows = state["read_key"].shape[0] - (case["tail"] if case["kind"] == "read" else 0)
    seq, pos = _places(state, starts, rows)
    page = state["pages"][seq, (pos // case["page"]).long()].long()
    slot = (pos % case["page"]).long()
    for name in ("key", "value"):
        x = state[name + "_cache"][page, :, slot]
        if case["cache"] == "int8":
            x = (x.float() * state[name + "_scales"][page, :, slot][..., None]).to(torch.bfloat16)
        state["read_" + name][:rows] = x


def _gathered(state, name):
    """Keys or values of every sequence, padded to the longest: [sequence, head, position, D] in 32 bits."""
    case = state["case"]
    if case["kind"] == "attention":
        starts, longest = state["row_starts"], _longest(case)
        at = (starts[:-1, None] + torch.arange(longest, device="cuda")).clamp_max(state[name].shape[0] - 1)
        return state[name][at].float().permute(0, 2, 1, 3)
    table = state["pages"].clamp_min(0).long()
    x = state[name + "_cache"][table].float()  # [sequence, page, head, slot, D]
    if case["cache"] == "int8":
        x *= state[name + "_scales"][table][..., None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attention(state):
    case = state["case"]
    S, H, KVH, D = case["S"], case["H"], case["KVH"], case["D"]
    starts, lengths = state["row_starts"], state["lengths"]
    n_max = max(n for n, _ in _sequences(case))
    n = starts[1:] - starts[:-1]
    row = torch.arange(n_max, device="cuda")
    at = (starts[:-1, None] + row).clamp_max(state["query"].shape[0] - 1)
    q = state["query"][at].float().reshape(S, n_max, KVH, H // KVH, D).permute(0, 2, 3, 1, 4).reshape(S, KVH, H // KVH * n_max, D)
    keys, values = _gathered(state, "key"), _gathered(state, "value")
    L = keys.shape[2]
    pos = (lengths - n)[:, None] + row  # [sequence, row]
    j = torch.arange(L, device="cuda")
    seen = j <= pos[..., None]
    if case["window"]:
        seen &= (j > pos[..., None] - case["window"]) | (j < case["sinks"])
    scores = torch.matmul(q, keys.transpose(2, 3)).mul_(_scale(case)).reshape(S, KVH, H // KVH, n_max, L)
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


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    page = case.get("page")
    starts, lengths = s["row_starts"].tolist(), s["lengths"].tolist()

    def slots(i, first, count):
        """Page and slot of `count` positions of sequence i."""
        p = torch.arange(first, first + count, device="cuda")
        return s["pages"][i].long()[p // page], p % page

    def held(i, name, codes=None, scales=None):
        """Keys or values of sequence i's positions: [position, head, D]."""
        if case["kind"] == "attention":
            return s[name][starts[i]:starts[i + 1]].double()
        g, o = slots(i, 0, lengths[i])
        x = (s[name + "_cache"] if codes is None else codes)[g, :, o].double()
        if case["cache"] == "int8":
            x = x * (s[name + "_scales"] if scales is None else scales)[g, :, o].double()[..., None]
        return x

    if case["kind"] in ("write", "append_read"):
        caches, sizes = [], []
        for name in ("key", "value"):
            cache = s[name + "_cache"].double()
            scales = s[name + "_scales"].double() if case["cache"] == "int8" else None
            for i in range(case["S"]):
                x = s[name][starts[i]:starts[i + 1]].double()
                g, o = slots(i, lengths[i] - x.shape[0], x.shape[0])
                if scales is None:
                    cache[g, :, o] = x
                else:
                    unit = x.abs().max(dim=-1).values.clamp(min=2.0 ** -100) / 127
                    scales[g, :, o] = unit
                    cache[g, :, o] = torch.round(x / unit[..., None])
            caches.append(cache)
            sizes.append(scales)
        if case["kind"] == "write":
            return caches
        back = [torch.cat([held(i, name, c, u) for i in range(case["S"])]) for name, c, u in zip(("key", "value"), caches, sizes)]
        return back + sizes
    if case["kind"] == "read":
        return [torch.cat([held(i, name) for i in range(case["S"])] + [s["read_" + name][starts[-1]:].double()]) for name in ("key", "value")]
    out, G = s["out"].double(), case["H"] // case["KVH"]
    for i in range(case["S"]):
        q, keys, values = s["query"][starts[i]:starts[i + 1]].double(), held(i, "key"), held(i, "value")
        n, L = q.shape[0], keys.shape[0]
        p, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
        for h in range(case["KVH"]):
            for g in range(h * G, h * G + G):
                weights = (q[:, g] @ keys[:, h].T / math.sqrt(case["D"])).masked_fill(hidden, -math.inf)
                out[starts[i]:starts[i + 1], g] = torch.softmax(weights, dim=-1) @ values[:, h]
    return out
