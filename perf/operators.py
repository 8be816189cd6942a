"""The operators of the quantised KV cache, case by case: writing rows into pages, reading them back, attention of new
tokens (one per sequence, a drafted tree, a causal chunk) over the pages, and keeping the accepted drafts of a tree.

A cache is two page pools (keys, values) of [pages, page_size, heads, head_dim] codes -- fp8 E4M3 / E5M2, fp4 E2M1 (two
codes a byte, the even element in the low half) or the 16-bit values themselves -- and, for the 8- and 4-bit formats,
two pools of power-of-two scales, uint8 [pages, heads, head_dim / group, page_size]: byte e stands for 2 ** (e - 127)
and belongs to `group` consecutive elements of a row.  A row's group is scaled by the smallest power of two that brings
its largest magnitude to the format's largest value or below, then rounded to nearest even.  A block table gives the
pages of a sequence; the new tokens of a sequence are its last ones.
"""
import math

import numpy as np
import torch

own = False

FORMATS = {"bf16": 0, "fp16": 1, "fp8_e4m3": 2, "fp8_e5m2": 3, "fp4_e2m1": 4}  # the package's HF_KV_* values
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FLOAT8 = {"fp8_e4m3": torch.float8_e4m3fn, "fp8_e5m2": torch.float8_e5m2}
# largest value of a format as mantissa (in [1, 2)) and exponent
LARGEST = {"fp8_e4m3": (1.75, 8), "fp8_e5m2": (1.75, 15), "fp4_e2m1": (1.5, 2)}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # serving, one new token of each of 64 conversations (Llama-3-8B's 8 KV heads of 128, 16-token pages)
        dict(name="write tokens", op="write", fmt="fp8_e4m3", dtype="bf16", batch=64, new=1, spread=0, past=1000, page=16,
             heads=8, dim=128, group=128),
        # a prompt pass over 16 ragged prompts
        dict(name="write prompts", op="write", fmt="fp8_e4m3", dtype="bf16", batch=16, new=4001, spread=1, past=0, page=16,
             heads=8, dim=128, group=128),
        # prompts into a 4-bit cache and back, to see what attention will see of them
        dict(name="write and read fp4", op="through", fmt="fp4_e2m1", dtype="fp16", batch=5, new=1777, spread=1, past=100,
             page=32, heads=4, dim=64, group=32),
        # a cache handed to something that takes 16-bit rows (another engine, a check against recomputed rows)
        dict(name="read contexts", op="read", fmt="fp8_e4m3", dtype="bf16", batch=32, new=2048, spread=1, past=0, page=16,
             heads=8, dim=128, group=128),
        # one conversation's rows, odd sizes
        dict(name="read one", op="read", fmt="fp8_e5m2", dtype="fp32", batch=1, new=1003, spread=0, past=0, page=8,
             heads=3, dim=96, group=32),
        # speculative decoding: write a tree of drafts, then keep the accepted path
        dict(name="keep of many", op="keep", fmt="fp8_e4m3", dtype="bf16", batch=64, new=48, spread=1, past=1500, page=16,
             heads=8, dim=128, group=128),
        dict(name="keep of one", op="keep", fmt="fp8_e5m2", dtype="bf16", batch=1, new=16, spread=0, past=700, page=16,
             heads=8, dim=128, group=32),
        # decoding one conversation: the smallest call, latency is all
        dict(name="attend one token", op="attend", fmt="fp8_e4m3", dtype="bf16", batch=1, new=1, spread=0, past=1000, page=16,
             heads=8, per=4, dim=128, group=128, tree=0),
        # decoding a batch of ragged conversations
        dict(name="attend tokens", op="attend", fmt="fp8_e4m3", dtype="bf16", batch=64, new=1, spread=0, past=8000, page=16,
             heads=8, per=4, dim=128, group=128, tree=0),
        # verifying drafted trees of a batch
        dict(name="attend trees", op="attend", fmt="fp8_e4m3", dtype="bf16", batch=8, new=63, spread=1, past=8000, page=16,
             heads=8, per=4, dim=128, group=128, tree=1),
        # verifying one tree over a long context in a 4-bit cache
        dict(name="attend tree, long", op="attend", fmt="fp4_e2m1", dtype="fp16", batch=1, new=29, spread=0, past=131000,
             page=64, heads=8, per=4, dim=128, group=32, tree=1),
        # a chunk of a prompt over what is cached, 16-bit cache
        dict(name="attend chunk", op="attend", fmt="bf16", dtype="bf16", batch=2, new=1000, spread=0, past=5000, page=16,
             heads=8, per=4, dim=128, group=0, tree=0),
    ]


def draw(rng):
    def between(lo, hi):  # spread over the logarithm, odd sizes as they fall
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["write", "through", "read", "keep", "attend", "attend", "attend"])
    fmt = rng.choice(["fp8_e4m3", "fp8_e4m3", "fp8_e5m2", "fp4_e2m1", "fp4_e2m1", "bf16", "fp16"])
    if fmt == "fp4_e2m1" and op in ("write", "keep"):
        op = "through"  # two 4-bit codes share a byte: they are looked at as what is read back
    dtype = fmt if fmt in DTYPES else rng.choice(["bf16", "fp16"])
    c = dict(op=op, fmt=fmt, dtype=dtype, page=rng.choice([8, 16, 32, 64, 128]), dim=rng.choice([64, 96, 128, 128, 256]))
    c["group"] = 0 if fmt in DTYPES else rng.choice([g for g in (32, 64, 128, 256) if c["dim"] % g == 0])
    c["heads"] = rng.choice([1, 2, 3, 4, 8, 8]) if c["dim"] < 256 else rng.choice([1, 2, 4])
    c["spread"] = rng.choice([0, 1])
    if op == "attend":
        kind = rng.choice(["token", "tree", "chunk"])
        c["per"] = rng.choice([1, 2, 4, 5, 8])
        c["tree"] = int(kind == "tree")
        c["batch"] = between(1, 64) if kind == "token" else between(1, 8)
        c["new"] = 1 if kind == "token" else between(2, 64) if kind == "tree" else between(16, 700)
        c["past"] = between(1, max(2, min(40000, 400000 // (c["batch"] * max(1, c["new"] // 64)))))
    elif op == "keep":
        c.update(batch=between(1, 64), new=between(2, 64), past=between(1, 2000))
    else:
        c["batch"] = between(1, 64)
        c["new"] = between(1, max(2, 60000 // c["batch"]))
        c["past"] = 0 if op == "read" else between(1, 500)
    return c


def _sizes(c):
    """New tokens and all tokens of each sequence, from the case alone: a ragged batch has lengths between a quarter of
    the case's and the whole, the first one the whole."""
    r = np.random.RandomState(len(c["op"]) + c["batch"] * 7 + c["new"] * 31 + c["past"] * 131)
    new, past = np.full(c["batch"], c["new"]), np.full(c["batch"], c["past"])
    if c["spread"]:
        new = np.maximum(1, (new * r.uniform(0.25, 1.0, c["batch"])).astype(int))
        new[0] = c["new"]
    if c["batch"] > 1:
        past = (past * r.uniform(0.25, 1.0, c["batch"])).astype(int)
        past[0] = c["past"]
    return new.astype(np.int64), (new + past).astype(np.int64)


def _code_bytes(c):
    """Bytes of one row of one head: codes and scales."""
    bits = {"bf16": 16, "fp16": 16, "fp8_e4m3": 8, "fp8_e5m2": 8, "fp4_e2m1": 4}[c["fmt"]]
    return c["dim"] * bits // 8 + (c["dim"] // c["group"] if c["group"] else 0)


def work(c):
    new, total = _sizes(c)
    n, h, d = int(new.sum()), c["heads"], c["dim"]
    size = 4 if c["dtype"] == "fp32" else 2
    wide, code = 2 * n * h * d * size, 2 * n * h * _code_bytes(c)
    if c["op"] in ("write", "read"):
        return {"bytes": wide + code, "flops": 0}
    if c["op"] == "through":  # rows in, codes out, codes in, rows out
        return {"bytes": 2 * wide + 2 * code, "flops": 0}
    if c["op"] == "keep":  # rows in, codes out, the kept half moved
        return {"bytes": wide + 2 * code, "flops": 0}
    seen = int(((total - new) * new).sum())  # every new token sees all of the past
    seen += n if c["tree"] else int((new * (new + 1) // 2).sum())  # and of the new ones at least itself
    rows = n * h * c["per"]
    return {"bytes": 2 * int(total.sum()) * h * _code_bytes(c) + rows * (2 * d * 2 + 4),
            "flops": 4 * d * h * c["per"] * seen}


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = np.random.RandomState(seed)
    new, total = _sizes(c)
    pages = -(-total // c["page"])
    width, count = int(pages.max()), int(pages.sum())
    order = r.permutation(count)
    table, at = np.zeros((c["batch"], width), np.int32), 0
    for b, k in enumerate(pages):
        table[b, :k] = order[at:at + k]
        at += int(k)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    h, d, dtype = c["heads"], c["dim"], DTYPES[c["dtype"]]

    def rows(n, heads, spread=1.0):
        # activations: channels of different size, as keys and values have them
        x = torch.randn(n, heads, d, generator=g, device="cuda")
        x *= torch.exp(0.7 * torch.randn(heads, d, generator=g, device="cuda")) * spread
        return x.to(DTYPES["bf16" if dtype == torch.float32 else c["dtype"]])

    s = dict(case=c, table=torch.from_numpy(table).cuda(), kv_len=torch.from_numpy(total.astype(np.int32)).cuda(),
             cu=torch.from_numpy(cu).cuda(), total=int(new.sum()), max_new=int(new.max()))
    s["batch_of"] = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), torch.from_numpy(new).cuda())
    # the pools hold what earlier calls wrote
    for name in ("k", "v"):
        codes, scales = [], []
        for lo in range(0, count * c["page"], 1 << 17):
            n = min(1 << 17, count * c["page"] - lo)
            q, e = _quantise(rows(n, h), c["fmt"], c["group"])
            codes.append(q)
            scales.append(e)
        s[name] = torch.cat(codes).view(count, c["page"], h, -1)
        if c["group"]:
            s[name + "_scale"] = torch.cat(scales).view(count, c["page"], h, -1).permute(0, 2, 3, 1).contiguous()
    if c["op"] in ("write", "through", "keep"):
        s["new_k"], s["new_v"] = rows(s["total"], h), rows(s["total"], h)
    if c["op"] == "attend":
        s["q"] = rows(s["total"], h * c["per"], 0.5)
        if c["tree"]:  # every draft continues an earlier one, or the past
            words = -(-s["max_new"] // 32)
            mask = np.zeros((s["total"], words), np.uint32)
            for b in range(c["batch"]):
                for i in range(int(new[b])):
                    if i:
                        p = int(r.randint(max(0, i - 8), i + 1)) - 1
                        if p >= 0:
                            mask[cu[b] + i] = mask[cu[b] + p]
                    mask[cu[b] + i, i // 32] |= np.uint32(1 << (i % 32))
            s["mask"] = torch.from_numpy(mask.view(np.int32)).cuda()
    if c["op"] == "keep":  # an accepted path of about half of the drafts, ascending
        path, length = np.zeros((c["batch"], s["max_new"]), np.int32), np.zeros(c["batch"], np.int32)
        for b in range(c["batch"]):
            keep = np.flatnonzero(r.uniform(size=int(new[b])) < 0.5)
            path[b, :len(keep)], length[b] = keep, len(keep)
        s["path"], s["path_len"] = torch.from_numpy(path).cuda(), torch.from_numpy(length).cuda()
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _two_to(e):
    """2 ** e of whole numbers in -126..127, exactly (a power function may be off by a last bit)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, fmt, group):
    """Codes (a byte tensor, or the 16-bit values) and scale bytes of rows [n, heads, dim]."""
    if fmt in DTYPES:
        return x.to(DTYPES[fmt]), None
    n, h, d = x.shape
    y = x.float().view(n, h, d // group, group)
    top = y.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    mant, power = LARGEST[fmt]
    e = e - 1 - power + (2 * m > mant).int()
    e = torch.where(top == 0, torch.zeros_like(e), e.clamp(min=-126))
    y = y * _two_to(-e)
    if fmt == "fp4_e2m1":
        a = y.abs()
        code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
                + (a >= 3.5).byte() + (a > 5.0).byte()) | (torch.signbit(y).byte() << 3)
        code = code.view(n, h, d // 2, 2)
        code = code[..., 0] | (code[..., 1] << 4)
    else:
        code = y.to(FLOAT8[fmt]).view(torch.uint8).view(n, h, d)
    return code, (e + 127).byte().view(n, h, d // group)


def _values(code, scale, fmt, group):
    """The values of codes [..., bytes] with scale bytes [..., groups], in 32 bits."""
    if fmt in DTYPES:
        return code.float()
    if fmt == "fp4_e2m1":
        both = torch.stack([code & 15, code >> 4], -1).flatten(-2)
        y = torch.tensor(FP4 + tuple(-a for a in FP4), device=code.device)[both.int()]
    else:
        y = code.view(FLOAT8[fmt]).float()
    return (y.unflatten(-1, (-1, group)) * _two_to(scale.int() - 127).unsqueeze(-1)).flatten(-2)


def _place(s):
    """Page and offset of each new token."""
    c, b = s["case"], s["batch_of"]
    i = torch.arange(s["total"], device="cuda") - s["cu"][b]
    pos = (s["kv_len"] - (s["cu"][1:] - s["cu"][:-1]))[b] + i
    return s["table"][b, pos // c["page"]].long(), (pos % c["page"]).long()


def _plain_write(s):
    c = s["case"]
    page, off = _place(s)
    for name in ("k", "v"):
        code, scale = _quantise(s["new_" + name], c["fmt"], c["group"])
        s[name][page, off] = code
        if c["group"]:
            s[name + "_scale"][page, :, :, off] = scale


def _plain_read(s):
    c = s["case"]
    page, off = _place(s)
    return tuple(_values(s[name][page, off], s[name + "_scale"][page, :, :, off] if c["group"] else None, c["fmt"], c["group"])
                 .to(DTYPES[c["dtype"]]) for name in ("k", "v"))


def _plain_keep(s):
    # the accepted drafts move to the first places behind the past
    c = s["case"]
    past = s["kv_len"] - (s["cu"][1:] - s["cu"][:-1])
    j = torch.arange(s["path"].shape[1], device="cuda")
    b, j = torch.nonzero(j < s["path_len"].unsqueeze(1), as_tuple=True)
    src, dst = past[b] + s["path"][b, j], past[b] + j
    sp, so = s["table"][b, src // c["page"]].long(), (src % c["page"]).long()
    dp, do = s["table"][b, dst // c["page"]].long(), (dst % c["page"]).long()
    for name in ("k", "v"):
        s[name][dp, do] = s[name][sp, so]
        if c["group"]:
            s[name + "_scale"][dp, :, :, do] = s[name + "_scale"][sp, :, :, so]
    return past + s["path_len"]


def _plain_attend(s):
    c = s["case"]
    batch, h, per, d, most = c["batch"], c["heads"], c["per"], c["dim"], s["max_new"]
    cap = s["table"].shape[1] * c["page"]
    pages = s["table"].long()

    def dense(name):  # [batch, heads, cap, dim]
        scale = s[name + "_scale"][pages].permute(0, 1, 4, 2, 3) if c["group"] else None
        return _values(s[name][pages], scale, c["fmt"], c["group"]).view(batch, cap, h, d).transpose(1, 2)

    n = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(most, device="cuda")
    row = (s["cu"][:-1, None] + i).clamp(max=s["total"] - 1).long()  # [batch, most]
    q = s["q"].float()[row].view(batch, most, h, per, d).permute(0, 2, 3, 1, 4).reshape(batch, h, per * most, d)
    score = torch.matmul(q, dense("k").transpose(2, 3)).view(batch, h, per, most, cap) / math.sqrt(d)
    t = torch.arange(cap, device="cuda")
    past = s["kv_len"] - n
    if c["tree"]:
        bits = ((s["mask"][row][..., None] >> torch.arange(32, device="cuda")) & 1).bool().flatten(2)  # [batch, most, drafts]
        draft = (t - past[:, None]).clamp(0, bits.shape[2] - 1)
        seen = bits.gather(2, draft[:, None].expand(-1, most, -1).long())
    else:
        seen = t - past[:, None, None] <= i[:, None]
    seen = ((t < past[:, None])[:, None] | seen) & (t < s["kv_len"][:, None])[:, None]
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, h, per * most, cap), dense("v")).view(batch, h, per, most, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + torch.log(total)).squeeze(-1)
    b, at = s["batch_of"], torch.arange(s["total"], device="cuda") - s["cu"][s["batch_of"]]
    out = out.permute(0, 3, 1, 2, 4)[b, at].reshape(s["total"], h * per, d)
    return out.to(DTYPES[c["dtype"]]), lse.permute(0, 3, 1, 2)[b, at].reshape(s["total"], h * per)


# ---- the package's calls -------------------------------------------------------------------------------------------
def _cache(s):
    """The handle that a user's program keeps beside its pools."""
    if "cache" not in s:
        from huffman_amd import KvCache
        s["cache"] = KvCache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"), fmt=FORMATS[s["case"]["fmt"]])
    return s["cache"]


def _own(s):
    c, cache = s["case"], _cache(s)
    one = s["max_new"] == 1  # one new token of each sequence: no list of row offsets is needed
    cu = None if one else s["cu"]
    if c["op"] in ("write", "through", "keep"):
        cache.write(s["new_k"], s["new_v"], s["table"], s["kv_len"], cu)
    if c["op"] in ("through", "read"):
        return cache.read(s["table"], s["kv_len"], cu, rows=s["total"], dtype=DTYPES[c["dtype"]])
    if c["op"] == "keep":
        return cache.keep(s["table"], s["kv_len"], cu, s["path"], s["path_len"])
    if c["op"] == "attend":
        return cache.attend(s["q"], s["table"], s["kv_len"], cu, max_q=s["max_new"], mask=s.get("mask"), lse=True)


def run(s):
    c = s["case"]
    if own:
        got = _own(s)
    else:
        if c["op"] in ("write", "through", "keep"):
            _plain_write(s)
        got = _plain_read(s) if c["op"] in ("through", "read") else _plain_keep(s) if c["op"] == "keep" \
            else _plain_attend(s) if c["op"] == "attend" else None
    if c["op"] in ("through", "read"):
        return {"k": got[0], "v": got[1]}
    if c["op"] == "attend":
        return {"out": got[0], "lse": got[1]}
    out = {"kv_len": got} if c["op"] == "keep" else {}
    for name in ("k", "v"):  # the pools, 8-bit codes as the values they stand for
        out[name] = s[name].view(FLOAT8[c["fmt"]]) if c["fmt"] in FLOAT8 else s[name]
        if c["group"]:
            out[name + "_scale"] = s[name + "_scale"]
    return out


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def _power(e):
    """2 ** e of whole numbers, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _grid(fmt):
    """Every value of a format that is not negative, ascending (index = code)."""
    if fmt == "fp4_e2m1":
        return torch.tensor(FP4, dtype=torch.float64, device="cuda")
    bits, bias = {"fp8_e4m3": (3, 7), "fp8_e5m2": (2, 15)}[fmt]
    last = {"fp8_e4m3": 126, "fp8_e5m2": 123}[fmt]
    v = []
    for code in range(last + 1):
        e, m = code >> bits, code & ((1 << bits) - 1)
        v.append((m if e == 0 else m + (1 << bits)) * 2.0 ** (max(e, 1) - bias - bits))
    return torch.tensor(v, dtype=torch.float64, device="cuda")


def _rounded(x, fmt, group):
    """Rows [n, heads, dim] as a cache of the format holds them, in 64 bits: (codes' values, scale exponents)."""
    x = x.double()
    if fmt in DTYPES:
        return x, None
    grid = _grid(fmt)
    y = x.unflatten(-1, (-1, group))
    top = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / grid[-1])).clamp(min=-126)
    e = torch.where(top > grid[-1] * _power(e), e + 1, e)  # the logarithm may be off by one
    e = torch.where((top <= grid[-1] * _power(e - 1)) & (e > -126), e - 1, e)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    a = (y * _power(-e)).abs()
    hi = torch.searchsorted(grid, a.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    down, up = a - grid[lo], grid[hi] - a
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(grid[code], y).flatten(-2), e.squeeze(-1)


def exact(c, seed):
    s = prepare(c, seed)
    new, total = _sizes(c)
    cu = np.concatenate([[0], np.cumsum(new)])

    def pages(b, lo, hi):
        t = torch.arange(int(lo), int(hi), device="cuda")
        return s["table"][b].long()[t // c["page"]], t % c["page"]

    def stored(name, b, lo, hi):  # rows lo..hi of a sequence out of the pool
        p, o = pages(b, lo, hi)
        code = s[name][p, o]
        if c["fmt"] in DTYPES:
            return code.double()
        if c["fmt"] == "fp4_e2m1":
            grid = torch.cat([_grid(c["fmt"]), -_grid(c["fmt"])])
            y = grid[torch.stack([code & 15, code >> 4], -1).flatten(-2).long()]
        else:
            y = code.view(FLOAT8[c["fmt"]]).double()
        e = s[name + "_scale"][p, :, :, o].double() - 127
        return (y.unflatten(-1, (-1, c["group"])) * _power(e).unsqueeze(-1)).flatten(-2)

    if c["op"] == "through":
        got = {}
        for name in ("k", "v"):
            y, e = _rounded(s["new_" + name], c["fmt"], c["group"])
            got[name] = y if e is None else (y.unflatten(-1, (-1, c["group"])) * _power(e).unsqueeze(-1)).flatten(-2)
        return got
    if c["op"] == "read":
        return {name: torch.cat([stored(name, b, total[b] - new[b], total[b]) for b in range(c["batch"])]) for name in ("k", "v")}
    if c["op"] in ("write", "keep"):
        got = {"kv_len": None} if c["op"] == "keep" else {}
        for name in ("k", "v"):
            if c["group"]:
                got[name + "_scale"] = None
            y, _ = _rounded(s["new_" + name], c["fmt"], c["group"])
            pool = s[name].view(FLOAT8[c["fmt"]]).double() if c["fmt"] in FLOAT8 else s[name].double()
            for b in range(c["batch"]):
                past = total[b] - new[b]
                p, o = pages(b, past, total[b])
                pool[p, o] = y[cu[b]:cu[b + 1]]
                if c["op"] == "keep":
                    n = int(s["path_len"][b])
                    path = s["path"][b, :n].long()
                    dp, do = pages(b, past, past + n)
                    pool[dp, do] = y[cu[b]:cu[b + 1]][path]
            got[name] = pool
        return got
    out, lse = [], []
    for b in range(c["batch"]):
        n, past = int(new[b]), int(total[b] - new[b])
        k, v = stored("k", b, 0, total[b]).transpose(0, 1), stored("v", b, 0, total[b]).transpose(0, 1)
        q = s["q"][cu[b]:cu[b + 1]].double().view(n, c["heads"], c["per"], c["dim"])
        seen = torch.ones(n, int(total[b]), dtype=torch.bool, device="cuda")
        if c["tree"]:
            words = s["mask"][cu[b]:cu[b + 1]].cpu().numpy().view(np.uint32)
            seen[:, past:] = torch.from_numpy(((words[:, np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1) > 0).cuda()
        else:
            seen[:, past:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        o = torch.empty(n, c["heads"], c["per"], c["dim"], dtype=torch.float64, device="cuda")
        z = torch.empty(n, c["heads"], c["per"], dtype=torch.float64, device="cuda")
        for h in range(c["heads"]):
            for j in range(c["per"]):
                w = (q[:, h, j] @ k[h].T) / math.sqrt(c["dim"])
                w = w.masked_fill(~seen, float("-inf"))
                z[:, h, j] = torch.logsumexp(w, -1)
                o[:, h, j] = torch.softmax(w, -1) @ v[h]
        out.append(o.view(n, -1, c["dim"]))
        lse.append(z.view(n, -1))
    return {"out": torch.cat(out), "lse": torch.cat(lse)}
