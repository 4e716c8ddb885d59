"""The operators a server over one packed page pool needs besides append and plain decode, as cases that can be timed and checked.

Three operators on the k2b cache (128-token pages in row order: low-rank fp16 coefficients + 3-bit residual nibbles for keys, 2-bit
codes under a Hadamard rotation for values, a recent window in fp16):

* "copy"     slots of the page pools or rows of the windows to other slots: fork, compaction, growth of a pool;
* "shared"   a decode step of sequences that share a long prefix of pages, which is read once for all of them;
* "slide"    attention with a sliding window and a few first tokens that stay visible, for single tokens ("slide_decode") and for
             blocks of prompt rows ("slide_prompt"); pages that no row sees are gone from the pool.

The plain forms are elementary torch operations in float32; `exact` restates the definitions in float64 with the index formulas of
the page layout.  Where `own` is true, `run` calls the library.
"""

import math

import torch

own = False

D = 128
PAGE = 128
RECENT = 128          # recent tokens that are never quantized
THETA = 5e5           # rotary base of the benchmark's model shape
LLOYD = (-1.5194618701934814, -0.46033763885498047, 0.44421979784965515, 1.5017313957214355)  # 2-bit levels of N(0, 1)
SCALE = 1.0 / math.sqrt(D)

HEADS = {"h_kv": 8, "q_groups": 4}
K2B = {**HEADS, "rank": 32, "group": 64, "shared_basis": False}


def listed():
    return [
        # a request sampled four ways: the fp16 window rows of the parent go to three more sequences (pages are shared, not copied)
        {"name": "copy_fork3_tail200", "kind": "copy", "what": "windows", "rows": 8, "copies": 3, "tail": 200, **K2B},
        # holes left by finished sequences are closed: 640 live slots move to the front of a pool of 2048
        {"name": "copy_compact_640", "kind": "copy", "what": "compact", "slots": 2048, "moved": 640, **K2B},
        # a full pool of 3000 slots is taken over by a larger one
        {"name": "copy_grow_3000", "kind": "copy", "what": "grow", "slots": 4096, "moved": 3000, **K2B},
        # four answers to one 8k-token document
        {"name": "shared_b4_t8192", "kind": "shared", "groups": 1, "members": 4, "prefix_pages": 64, "own_tokens": 300, **K2B},
        # 32 requests over one 32k-token system prompt and document
        {"name": "shared_b32_t32768", "kind": "shared", "groups": 1, "members": 32, "prefix_pages": 256, "own_tokens": 600, **K2B},
        # three documents of 5k tokens with 21 questions each, one basis over all heads, two KV heads with eight query heads
        {"name": "shared_g3x21_t5120", "kind": "shared", "groups": 3, "members": 21, "prefix_pages": 40, "own_tokens": 450, "h_kv": 2, "q_groups": 8,
         "rank": 16, "group": 32, "shared_basis": True},
        # 128 short chats behind one 16k-token prefix
        {"name": "shared_b128_t16384", "kind": "shared", "groups": 1, "members": 128, "prefix_pages": 128, "own_tokens": 200, **K2B},
        # one user, far into a conversation that keeps 1024 tokens and four sinks
        {"name": "slide_b1_w1024", "kind": "slide_decode", "batch": 1, "tokens": 32768 + 128, "window": 1024, "sinks": 4, **K2B},
        # sixteen sequences of up to 16k tokens under a window of 4096
        {"name": "slide_b16_w4096", "kind": "slide_decode", "batch": 16, "tokens": 16384 + 128, "window": 4096, "sinks": 4, **K2B},
        # ragged and odd: shorter than the window some of them, sinks that end inside the second page
        {"name": "slide_b5_w777", "kind": "slide_decode", "batch": 5, "tokens": 2900, "window": 777, "sinks": 130, "h_kv": 3, "q_groups": 2,
         "rank": 16, "group": 128, "shared_basis": True},
        # a follow-up turn of 512 tokens far into a long conversation
        {"name": "slide_prompt_n512_w4096", "kind": "slide_prompt", "batch": 1, "rows": 512, "tokens": 32768 + 128, "window": 4096, "sinks": 4, **K2B},
        # a block of 2048 rows of two prompts
        {"name": "slide_prompt_n2048_w2048", "kind": "slide_prompt", "batch": 2, "rows": 2048, "tokens": 8192 + 128, "window": 2048, "sinks": 4, **K2B},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["copy", "shared", "shared", "slide_decode", "slide_decode", "slide_prompt"])
    rank, group = rng.choice([16, 32]), rng.choice([32, 64, 128])
    case = {"kind": kind, "h_kv": rng.choice([1, 2, 3, 4, 8]), "q_groups": rng.choice([1, 2, 4, 8]), "rank": rank, "group": group,
            "shared_basis": rng.random() < 0.4}
    if kind == "copy":
        case["what"] = rng.choice(["windows", "compact", "grow"])
        if case["what"] == "windows":
            case.update(rows=rng.choice([8, 16, 40]), tail=rng.randint(1, 2 * RECENT - 1))
            case["copies"] = rng.randint(1, case["rows"] - 1)
        else:
            case["moved"] = _log(rng, 1, 2400 if case["what"] == "grow" else 1000)
            case["slots"] = 2 * case["moved"] + rng.randint(0, 50)
    elif kind == "shared":
        case["groups"] = rng.choice([1, 1, 2, 3])
        case["prefix_pages"] = _log(rng, 1, 256 // case["groups"])
        case["members"] = _log(rng, 2, max(2, min(128, 32 * 256 // case["prefix_pages"]) // case["groups"]))
        case["own_tokens"] = _log(rng, 1, 1500)
    else:
        case["window"] = _log(rng, 1, 8192 if kind == "slide_decode" else 4096)
        case["sinks"] = rng.choice([0, 1, 4, 64, 129, 300])
        if kind == "slide_decode":
            case["batch"] = _log(rng, 1, max(1, min(32, 16 * 4096 // case["window"])))
            case["tokens"] = _log(rng, 1, 32768)
        else:
            case["rows"] = _log(rng, 1, 2048)
            case["batch"] = 1 if case["rows"] > 700 else rng.choice([1, 2, 3])
            case["tokens"] = case["rows"] + _log(rng, 1, 32768 - case["rows"])
            if case["rows"] > 1024:
                case["window"] = min(case["window"], 2048)
    return case


# ---- lengths -----------------------------------------------------------------------------------------------------------


def _held(tokens):
    """(committed pages, tokens in the fp16 window) of a sequence: whole pages beyond the recent window are packed."""
    pages = max(0, tokens - RECENT) // PAGE
    return pages, tokens - pages * PAGE


def _lengths(case):
    """(pages, tail) of every sequence; what a sequence holds behind a shared prefix, or in all."""
    if case["kind"] == "shared":
        n, most = case["groups"] * case["members"], case["own_tokens"]
        return [(case["prefix_pages"] + p, t) for p, t in (_held(1 + (i * 61 + most - 1) % most) for i in range(n))]
    if case["kind"] == "slide_prompt":
        return [_held(case["tokens"])] * case["batch"]
    return [_held(case["tokens"] - (i * 977) % max(1, case["tokens"] // 2)) for i in range(case["batch"])]


def _visible_pages(case):
    """(first pages kept for the sinks, first page of the window) of every sequence; pages between them are gone."""
    keep = -(-case["sinks"] // PAGE)
    out = []
    for pages, tail in _lengths(case):
        first_row = case["tokens"] - case["rows"] if "rows" in case else pages * PAGE + tail - 1
        out.append((min(keep, pages), min(pages, max(0, first_row - case["window"] + 1) // PAGE)))
    return out


# ---- seeded inputs -----------------------------------------------------------------------------------------------------


def _device():
    return torch.device("cuda") if torch.cuda.is_available() else torch.device("cpu")


def _block_bytes(case):
    return PAGE * 64 + PAGE // case["group"] * 256 + PAGE * 32 + PAGE * 2


def _coef_heads(case):
    return 1 if case["shared_basis"] else case["h_kv"]


def _pool(case, n, gen):
    """Random page blocks (n, h_kv, bytes) and coefficient blocks (n, coef heads, bytes) with the distributions the codec leaves:
    codes of a normal residual, scales of its group maximum, Gaussian value codes, norms of 128 normal values."""
    dev, h, r = gen.device, case["h_kv"], case["rank"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    nib = (normal(n, h, 2 * PAGE * 64) * 1.2).round_().clamp_(-4, 3).to(torch.int16).bitwise_and_(15).view(n, h, -1, 2)
    kres = (nib[..., 0] | (nib[..., 1] << 4)).to(torch.uint8)
    kscale = (normal(n, h, PAGE // case["group"] * D) * 0.2).exp_().mul_(0.08).half().view(torch.uint8)
    two = torch.bucketize(normal(n, h, 4 * PAGE * 32), torch.tensor([-0.99, 0.0, 0.97], device=dev)).to(torch.int16).view(n, h, -1, 4)
    vcode = (two[..., 0] | (two[..., 1] << 2) | (two[..., 2] << 4) | (two[..., 3] << 6)).to(torch.uint8)
    vnorm = (normal(n, h, PAGE) * 0.7 + math.sqrt(D)).half().view(torch.uint8)
    pages = torch.cat([kres, kscale, vcode, vnorm], -1).contiguous()
    decay = 6.0 * torch.arange(1, r + 1, device=dev).float() ** -0.75
    coef = normal(n, _coef_heads(case), 16, r // 8, 8, 8) * decay.view(1, 1, 1, r // 8, 1, 8)
    coefs = coef.half().reshape(n, _coef_heads(case), -1).view(torch.uint8)
    return pages, coefs.contiguous()


def _basis(case, gen):
    b = torch.stack([torch.linalg.qr(torch.randn(D, case["rank"], generator=gen, device=gen.device))[0] for _ in range(case["h_kv"])])
    return b.reshape(case["h_kv"] * D, case["rank"]).half().contiguous()


def _tables(n_pos, dev):
    inv = THETA ** (-torch.arange(0, D, 2, device=dev).double() / D)
    angle = torch.arange(n_pos, device=dev).double()[:, None] * inv
    angle = torch.cat([angle, angle], -1)
    return angle.cos().half(), angle.sin().half()


def _geom(case):
    from bmx_b200 import kernels as K

    return K.k2b_geom(case["h_kv"], case["q_groups"], PAGE, case["rank"], case["group"], _coef_heads(case))


def prepare(case, seed):
    gen = torch.Generator(device=_device()).manual_seed(int(seed))
    dev, h, H = gen.device, case["h_kv"], case["h_kv"] * case["q_groups"]
    host = torch.Generator().manual_seed(int(seed))
    s = {"case": case}
    if case["kind"] == "copy":
        return _prepare_copy(case, s, gen, host)
    held = _lengths(case)
    B = len(held)
    n_pages, tail = [p for p, _ in held], [t for _, t in held]
    width = max(1, max(n_pages))
    if case["kind"] == "shared":
        P, m = case["prefix_pages"], case["members"]
        used = [[(b // m) * P + j for j in range(P)] for b in range(B)]
        at = case["groups"] * P
        for b in range(B):
            used[b] += range(at, at + n_pages[b] - P)
            at += n_pages[b] - P
    else:
        used, at = [], 0
        for b, (keep, first) in enumerate(_visible_pages(case)):
            alive = [j for j in range(n_pages[b]) if j < keep or j >= first]
            row = [-1] * n_pages[b]
            for j in alive:
                row[j], at = at, at + 1
            used.append(row)
    n_slots = max(1, at)
    place = torch.randperm(n_slots, generator=host).to(torch.int32)       # slots of a sequence lie anywhere in the pool
    table = torch.full((B, width), -1, dtype=torch.int32)
    for b in range(B):
        ids = torch.tensor(used[b], dtype=torch.int64)
        table[b, : len(ids)] = torch.where(ids >= 0, place[ids.clamp(min=0)], -1)
    pages, coefs = _pool(case, n_slots, gen)
    cos, sin = _tables(width * PAGE + 2 * PAGE, dev)
    cap = RECENT + PAGE
    s.update(pages=pages, coefs=coefs, basis=_basis(case, gen), table=table.to(dev), n_pages=torch.tensor(n_pages, dtype=torch.int32, device=dev),
             tail_len=torch.tensor(tail, dtype=torch.int32, device=dev), max_pages=max(n_pages), cos=cos, sin=sin,
             k_tail=(torch.randn(B, h, cap, D, generator=gen, device=dev) * 0.6).half(), v_tail=torch.randn(B, h, cap, D, generator=gen, device=dev).half(),
             signs=(torch.randint(0, 2, (D,), generator=gen, device=dev) * 2 - 1).float())
    shape = (B, H, case["rows"], D) if "rows" in case else (B, H, D)
    s["q"] = torch.randn(*shape, generator=gen, device=dev).half()
    if own:
        from bmx_b200 import kernels as K

        g = _geom(case)
        pool = K.K2bPool(g, n_slots, dev)
        pool.pages.copy_(pages), pool.coefs.copy_(coefs)
        s.update(pool=pool, v_lut=K.v_lut_tensor(LLOYD, dev))
        if case["kind"] != "slide_decode":
            s["rope"] = K.rope_fragments(cos, sin, width + 1)
        if case["kind"] == "shared":
            m = case["members"]
            s["plan"] = K.PrefixGroups(g, B, [list(range(i * m, i * m + m)) for i in range(case["groups"])], [case["prefix_pages"]] * case["groups"], dev)
            s["workspace"] = K.decode_shared_workspace(g, B, s["plan"], dev)
        else:
            s["workspace"] = K.decode_workspace(g, B, s["max_pages"], dev)
    return s


def _prepare_copy(case, s, gen, host):
    h, dev = case["h_kv"], gen.device
    if case["what"] == "windows":
        cap, rows = RECENT + PAGE, case["rows"]
        order = torch.randperm(rows, generator=host).tolist()
        parent, children = order[0], order[1: 1 + case["copies"]]
        s["from_slots"] = [parent * h + i for _ in children for i in range(h)]
        s["to_slots"] = [c * h + i for c in children for i in range(h)]
        wins = [torch.randn(rows * h, cap, D, generator=gen, device=dev).half() for _ in range(3)]
        s["src"] = s["dst"] = [w[:, : case["tail"]] for w in wins]
        s["whole"] = wins
        return s
    n, moved = case["slots"], case["moved"]
    pages, coefs = _pool(case, n, gen)
    if case["what"] == "compact":
        holes = sorted(torch.randperm(n // 2, generator=host)[:moved].tolist())
        live = (n - 1 - torch.randperm(n - n // 2, generator=host)[:moved]).tolist()
        s.update(src=[pages, coefs], dst=[pages, coefs], from_slots=live, to_slots=holes)
    else:
        s.update(src=[pages, coefs], dst=[torch.zeros_like(pages), torch.zeros_like(coefs)],
                 from_slots=torch.randperm(n, generator=host)[:moved].tolist(), to_slots=list(range(moved)))
    s["whole"] = s["dst"]
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------


def _dequant(s, slots):
    """Page slots of any shape -> rotated-back values and pre-rotation keys, float32 (*slots, h_kv, 128 tokens, 128)."""
    case = s["case"]
    h, g, r = case["h_kv"], case["group"], case["rank"]
    flat = slots.reshape(-1).clamp(min=0).long()
    n = flat.numel()
    blk, cf = s["pages"][flat], s["coefs"][flat]
    dev = blk.device
    cuts = [PAGE * 64, PAGE // g * 256, PAGE * 32, PAGE * 2]
    kres, kscale, vcode, vnorm = torch.split(blk, cuts, -1)
    cc = torch.arange(8, device=dev)
    words = kres.contiguous().view(torch.int32).view(n, h, 4, PAGE, 2, 2, 1)                # chunk, token, upper half, octet
    code = (((words >> (16 * (cc & 1) + 4 * (cc >> 1))) & 15) ^ 8) - 8
    code = code.permute(0, 1, 3, 4, 2, 5, 6).reshape(n, h, PAGE // g, g, D).float()
    res = (code * kscale.contiguous().view(torch.float16).view(n, h, PAGE // g, 1, D).float()).view(n, h, PAGE, D)
    coef = cf.view(torch.float16).view(n, _coef_heads(case), 16, r // 8, 8, 8).transpose(3, 4).reshape(n, _coef_heads(case), PAGE, r).float()
    k = coef @ s["basis"].float().view(h, D, r).transpose(1, 2) + res
    tau = torch.arange(16, device=dev)
    shift = torch.where(tau < 8, 4 * tau, 4 * (tau - 8) + 2)
    words = vcode.contiguous().view(torch.int32).view(n, h, 2, D, 4, 1)
    idx = ((words >> shift) & 3).permute(0, 1, 2, 4, 5, 3).reshape(n, h, PAGE, D).long()
    lev = torch.tensor(LLOYD, device=dev)[idx]
    had = torch.ones(1, 1, device=dev)
    for _ in range(7):
        had = torch.cat([torch.cat([had, had], 1), torch.cat([had, -had], 1)], 0)
    v = (lev @ had) * (s["signs"] / D) * vnorm.contiguous().view(torch.float16).view(n, h, PAGE, 1).float()
    return k.view(*slots.shape, h, PAGE, D), v.view(*slots.shape, h, PAGE, D)


def _keys_values(s, slots, page_no):
    """Pages (batch, n) -> rotated keys and values (batch, h_kv, n * 128, 128) and the keys' positions (batch, n * 128)."""
    k, v = _dequant(s, slots)
    pos = (page_no[..., None] * PAGE + torch.arange(PAGE, device=slots.device)).long()
    at = pos.clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at].float().unsqueeze(2), s["sin"][at].float().unsqueeze(2)
    k = k * cos + torch.cat([-k[..., D // 2:], k[..., : D // 2]], -1) * sin
    b, n, h = k.shape[:3]
    return k.transpose(1, 2).reshape(b, h, n * PAGE, D), v.transpose(1, 2).reshape(b, h, n * PAGE, D), pos.view(b, n * PAGE)


def _softmax(scores, seen):
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), torch.zeros_like(top), top))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_shared(s):
    case, dev = s["case"], s["q"].device
    P, m, h = case["prefix_pages"], case["members"], case["h_kv"]
    B, H, _ = s["q"].shape
    G, T = H // h, P * PAGE
    heads = s["table"][::m, :P]
    kp, vp, _ = _keys_values(s, heads, torch.arange(P, device=dev).expand(heads.shape[0], P))      # once per group
    q = s["q"].float().view(-1, m, h, G, D).transpose(1, 2).reshape(-1, h, m * G, D)
    sp = ((q @ kp.transpose(2, 3)) * SCALE).view(-1, h, m, G, T).transpose(1, 2).reshape(B, h, G, T)
    mo = s["table"].shape[1] - P
    number = torch.arange(P, P + mo, device=dev).expand(B, mo)
    seen = [torch.ones(B, 1, 1, T, dtype=torch.bool, device=dev)]
    q = s["q"].float().view(B, h, G, D)
    ko, vo, pos = _keys_values(s, s["table"][:, P:], number)
    seen.append((pos < s["n_pages"][:, None] * PAGE).view(B, 1, 1, -1))
    kt, vt = s["k_tail"].float(), s["v_tail"].float()
    seen.append((torch.arange(kt.shape[2], device=dev) < s["tail_len"][:, None]).view(B, 1, 1, -1))
    scores = torch.cat([sp, (q @ ko.transpose(2, 3)) * SCALE, (q @ kt.transpose(2, 3)) * SCALE], -1)
    p = _softmax(scores, torch.cat(seen, -1))
    pp = p[..., :T].reshape(-1, m, h, G, T).transpose(1, 2).reshape(-1, h, m * G, T)
    out = (pp @ vp).view(-1, h, m, G, D).transpose(1, 2).reshape(B, h, G, D)
    own_end = T + mo * PAGE
    out = out + p[..., T:own_end] @ vo + p[..., own_end:] @ vt
    return out.reshape(B, H, D).half()


def _plain_slide(s):
    case, dev = s["case"], s["q"].device
    rows = case.get("rows", 1)
    q = s["q"].float().view(s["q"].shape[0], case["h_kv"], case["q_groups"] * rows, D)
    B, h = q.shape[:2]
    n_pages, total = s["n_pages"].long(), (s["n_pages"] * PAGE + s["tail_len"]).long()
    row_pos = (total[:, None] - rows + torch.arange(rows, device=dev)).repeat(1, case["q_groups"]).view(B, 1, -1, 1)
    first = ((total - rows - case["window"] + 1).clamp(min=0) // PAGE).minimum(n_pages)
    keep = -(-case["sinks"] // PAGE)
    gap = (first - keep).clamp(min=0)
    j = torch.arange(_most_visible(case), device=dev).expand(B, -1)
    number = torch.where(j < keep, j, j + gap[:, None])
    inside = number < n_pages[:, None]
    slots = s["table"].gather(1, number.clamp(max=s["table"].shape[1] - 1)) if j.shape[1] else torch.zeros(B, 0, dtype=torch.int32, device=dev)
    k, v, pos = _keys_values(s, slots, number)
    pos = torch.where(inside.repeat_interleave(PAGE, 1), pos, torch.full_like(pos, 1 << 40))
    t = torch.arange(s["k_tail"].shape[2], device=dev)
    tail_pos = torch.where(t < s["tail_len"][:, None], n_pages[:, None] * PAGE + t, torch.full((1, 1), 1 << 40, device=dev))
    pos = torch.cat([pos, tail_pos], 1).view(B, 1, 1, -1)
    seen = (pos <= row_pos) & ((pos < case["sinks"]) | (pos > row_pos - case["window"]))
    k, v = torch.cat([k, s["k_tail"].float()], 2), torch.cat([v, s["v_tail"].float()], 2)
    out = _softmax((q @ k.transpose(2, 3)) * SCALE, seen) @ v
    return out.reshape(s["q"].shape).half()


def _most_visible(case):
    return max(max(0, pages - max(0, first - keep)) for (keep, first), (pages, _) in zip(_visible_pages(case), _lengths(case)))


def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    if case["kind"] == "copy":
        for src, dst in zip(s["src"], s["dst"]):
            dst[torch.tensor(s["to_slots"], device=dst.device)] = src[torch.tensor(s["from_slots"], device=src.device)]
        return s["whole"]
    return _plain_shared(s) if case["kind"] == "shared" else _plain_slide(s)


def _run_own(s):
    from bmx_b200 import kernels as K

    case = s["case"]
    if case["kind"] == "copy":
        K.copy_slots(s["src"], s["dst"], s["from_slots"], s["to_slots"])
        return s["whole"]
    if case["kind"] == "shared":
        return K.k2b_decode_shared(s["pool"], s["q"], s["basis"], s["table"], s["n_pages"], s["max_pages"], s["plan"], s["cos"], s["sin"], s["rope"],
                                   s["k_tail"], s["v_tail"], s["tail_len"], s["v_lut"], s["signs"], SCALE, s["workspace"])
    if case["kind"] == "slide_decode":
        return K.k2b_decode_sliding(s["pool"], s["q"], s["basis"], s["table"], s["n_pages"], s["max_pages"], s["cos"], s["sin"], s["k_tail"],
                                    s["v_tail"], s["tail_len"], s["v_lut"], s["signs"], SCALE, s["workspace"], case["window"], case["sinks"])
    return K.k2b_prefill_sliding(s["pool"], s["q"], case["tokens"] - case["rows"], s["basis"], s["table"], s["n_pages"], s["max_pages"], s["cos"], s["sin"],
                                 s["rope"], s["k_tail"], s["v_tail"], s["tail_len"], s["v_lut"], s["signs"], SCALE, s["workspace"], case["window"],
                                 case["sinks"])


# ---- what a pass cannot do without -------------------------------------------------------------------------------------


def _token_bytes(case):
    """Packed bytes of one token of one KV head (coefficients, residual codes and scales, value codes, norm)."""
    return 2 * case["rank"] * _coef_heads(case) / case["h_kv"] + D / 2 + 2 * D / case["group"] + D / 4 + 2


def work(case):
    h, G = case["h_kv"], case["q_groups"]
    if case["kind"] == "copy":
        if case["what"] == "windows":
            return {"bytes": (1 + case["copies"]) * 3 * h * case["tail"] * 2 * D, "flops": 0}
        return {"bytes": 2 * case["moved"] * (h * _block_bytes(case) + _coef_heads(case) * PAGE * case["rank"] * 2), "flops": 0}
    held = _lengths(case)
    rows = case.get("rows", 1)
    packed = fp16 = pairs = 0
    if case["kind"] == "shared":
        packed = case["groups"] * case["prefix_pages"] * PAGE
        for pages, tail in held:
            packed, fp16, pairs = packed + (pages - case["prefix_pages"]) * PAGE, fp16 + tail, pairs + pages * PAGE + tail
    else:
        for pages, tail in held:
            total, committed = pages * PAGE + tail, pages * PAGE
            first = max(0, total - rows - case["window"] + 1)               # first key that some row's window reaches
            reached = [p for p in (min(case["sinks"], first), total - first)]
            packed += min(case["sinks"], first, committed) + max(0, committed - first)
            fp16 += sum(reached) - (min(case["sinks"], first, committed) + max(0, committed - first))
            for x in range(total - rows, total):
                low = max(0, x - case["window"] + 1)
                pairs += x + 1 - low + min(case["sinks"], low)
    n = len(held)
    return {"bytes": h * (packed * _token_bytes(case) + fp16 * 4 * D) + 4 * n * rows * h * G * D, "flops": h * (pairs * G * 4 * D + packed * 2 * D * case["rank"])}


# ---- float64 restatement -----------------------------------------------------------------------------------------------


def _exact_pages(s, slots, numbers):
    """Keys rotated at their positions and values of the given page slots, float64 (h_kv, tokens, 128), by the index formulas."""
    case, dev = s["case"], s["pages"].device
    h, g, r = case["h_kv"], case["group"], case["rank"]
    t = torch.arange(PAGE, device=dev)[:, None]
    c = torch.arange(D, device=dev)[None, :]
    n = len(slots)
    if n == 0:
        return torch.zeros(h, 0, D, dtype=torch.float64, device=dev), torch.zeros(h, 0, D, dtype=torch.float64, device=dev)
    blk, cf = s["pages"][torch.tensor(slots, device=dev)], s["coefs"][torch.tensor(slots, device=dev)]
    # residual code of (token t, channel c): nibble (c & 7) / 2 of the half c & 1 of its word
    word = (((c & 63) >> 4) * PAGE + t) * 4 + 2 * (c >> 6) + ((c & 15) >> 3)
    bit = 16 * (c & 1) + 4 * ((c & 7) >> 1)
    byte = blk[:, :, (word * 4 + bit // 8).reshape(-1)].view(n, h, PAGE, D).int()
    code = (byte >> (bit % 8)) & 15
    code = torch.where(code > 7, code - 16, code).double()
    off = PAGE * 64
    scale = blk[:, :, off: off + PAGE // g * 256].contiguous().view(torch.float16).view(n, h, PAGE // g, D).double()
    off += PAGE // g * 256
    word = ((t >> 6) * D + c) * 4 + ((t & 63) >> 4)
    bit = 4 * (t & 7) + 2 * ((t & 15) >> 3)
    byte = blk[:, :, (off + word * 4 + bit // 8).reshape(-1)].view(n, h, PAGE, D).int()
    lev = torch.tensor(LLOYD, dtype=torch.float64, device=dev)[((byte >> (bit % 8)) & 3).long()]
    off += PAGE * 32
    norm = blk[:, :, off:].contiguous().view(torch.float16).view(n, h, PAGE).double()
    i = torch.arange(r, device=dev)[None, :]
    at = ((t // 8) * (r // 8) + i // 8) * 64 + (t % 8) * 8 + i % 8
    coef = cf.view(torch.float16).double()[:, :, at.reshape(-1)].view(n, -1, PAGE, r).expand(n, h, PAGE, r)
    k = torch.einsum("nhtr,hcr->nhtc", coef, s["basis"].double().view(h, D, r)) + scale[:, :, torch.arange(PAGE, device=dev) // g] * code
    pos = (torch.tensor(numbers, device=dev)[:, None] * PAGE + torch.arange(PAGE, device=dev)).view(n, 1, PAGE)
    cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]
    rot = torch.empty_like(k)
    rot[..., : D // 2] = k[..., : D // 2] * cos[..., : D // 2] - k[..., D // 2:] * sin[..., : D // 2]
    rot[..., D // 2:] = k[..., D // 2:] * cos[..., D // 2:] + k[..., : D // 2] * sin[..., D // 2:]
    x = torch.arange(D, device=dev)
    parity = torch.zeros(D, D, dtype=torch.int64, device=dev)
    for b in range(7):                                                    # Hadamard entry (i, j): (-1)^(bits that i and j share)
        parity ^= ((x[:, None] & x[None, :]) >> b) & 1
    v = (lev / math.sqrt(D)) @ ((1 - 2 * parity).double() / math.sqrt(D)) * s["signs"].double() * norm[..., None]
    return rot.transpose(0, 1).reshape(h, -1, D), v.transpose(0, 1).reshape(h, -1, D)


def exact(case, seed):
    """What `run` returns, in float64; copied page bytes have no computed numbers."""
    if case["kind"] == "copy" and case["what"] != "windows":
        return None
    s = prepare(case, seed)
    if case["kind"] == "copy":
        whole = [w.double() for w in s["whole"]]
        for w in whole:
            for a, b in zip(s["from_slots"], s["to_slots"]):
                w[b, : case["tail"]] = w[a, : case["tail"]]
        return whole
    h, G, rows, dev = case["h_kv"], case["q_groups"], case.get("rows", 1), s["q"].device
    table, out, prefix = s["table"].tolist(), [], {}
    for b, (pages, tail) in enumerate(_lengths(case)):
        if case["kind"] == "shared":
            P, group = case["prefix_pages"], b // case["members"]
            if group not in prefix:
                prefix[group] = _exact_pages(s, table[b][:P], list(range(P)))
            k, v = _exact_pages(s, table[b][P:pages], list(range(P, pages)))
            k, v = torch.cat([prefix[group][0], k], 1), torch.cat([prefix[group][1], v], 1)
            numbers = list(range(pages))
        else:
            numbers = [j for j in range(pages) if table[b][j] >= 0]
            k, v = _exact_pages(s, [table[b][j] for j in numbers], numbers)
        k, v = torch.cat([k, s["k_tail"][b, :, :tail].double()], 1), torch.cat([v, s["v_tail"][b, :, :tail].double()], 1)
        pos = torch.tensor([j * PAGE + t for j in numbers for t in range(PAGE)] + [pages * PAGE + t for t in range(tail)], device=dev)
        total = pages * PAGE + tail
        q = s["q"][b].double().view(h, G, rows, D)
        got = []
        for r0 in range(0, rows, 256):                                    # bounded score matrices
            x = torch.arange(total - rows + r0, total - rows + min(rows, r0 + 256), device=dev)[:, None]
            seen = pos <= x
            if "window" in case:
                seen &= (pos < case["sinks"]) | (x - pos < case["window"])
            sc = (torch.einsum("hgnd,htd->hgnt", q[:, :, r0:r0 + 256], k) / math.sqrt(D)).masked_fill(~seen, float("-inf"))
            got.append(torch.einsum("hgnt,htd->hgnd", torch.softmax(sc, -1), v))
        out.append(torch.cat(got, 2).reshape(h * G, rows, D))
    out = torch.stack(out)
    return out if "rows" in case else out[:, :, 0]
