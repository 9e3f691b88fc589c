"""Performance cases of the operators around a layer's cached attention.

What a program that serves a DSA layer calls for its new tokens and its 4-bit
caches, each in its plain form (elementary torch operations in float32) and,
with ``own`` set, as the calls of ``lagged_indexer_dsa_amd.ops``:

* ``norm``   -- RMS norm with the residual's addition, its output in the
  input's type or in e4m3 with a scale per 128 values or per row
  (``ops.rms_norm``, ``ops.rms_norm_quant``).
* ``rotary`` -- the position rotation of a slice of the queries, written to a
  slice of the attention's query tensor (``ops.rotary``).
* ``append`` -- latent rows (normed and rotated on the way) and index keys
  (rotated) of new tokens into the paged caches, the latent rows in 8 or 4
  bits (``ops.append_tokens``); 4-bit rows come back as the values they hold
  (``ops.read_latent_rows``).
* ``read``   -- cached latent rows as bf16 values, as a prompt's next chunk
  attends them (``ops.read_latent_rows``).
* ``sparse``, ``dense`` -- decode attention over the 4-bit latent cache:
  selected rows, or every row's whole prefix (``ops.sparse_mla_decode``,
  ``ops.dense_mla_decode``).

Ranges: 1-8191 tokens; rows of 64 to 18432 values, odd ones among them;
float32, bfloat16 and float16; 1-128 heads; positions up to 163839; 1-64
requests of 0-131072 cached tokens, top-64 to top-2048.

Latent rows: 656 bytes = 512 e4m3, 4 float32 scales (one per 128 values), 64
bf16; 400 bytes = 512 e2m1 (value 2i in the low half of byte i), 16 e8m0
scales (one per 32 values), 64 bf16.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 64
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
_CONST: dict = {}


# ---------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # a layer's entry for one new token: four tensors of 14 KB, all latency
        dict(name="norm_token", kind="norm", tokens=1, dim=7168, dtype="bfloat16", residual=True, quant="none", pad=0),
        # a prompt's tokens entering an fp8 projection (odd count)
        dict(name="norm_prompt_fp8", kind="norm", tokens=8191, dim=7168, dtype="bfloat16", residual=True, quant="128",
             pad=0),
        # the rotary slice of a decode batch's queries, one tensor-parallel share of heads
        dict(name="rotary_batch", kind="rotary", tokens=32, heads=16, nope=128, rot=64, dtype="bfloat16",
             interleaved=True, inverse=False, max_pos=131072, yarn=True),
        # the same for a prompt and all heads (odd count)
        dict(name="rotary_prompt", kind="rotary", tokens=4097, heads=128, nope=128, rot=64, dtype="bfloat16",
             interleaved=True, inverse=False, max_pos=131072, yarn=True),
        # one new token of one request, 8-bit caches
        dict(name="append_token", kind="append", rows=1, tokens=1, start=5000, bits=8, dtype="bfloat16", norm=True,
             keys=True, interleaved=True, max_pos=131072),
        # a prompt's tokens into the 4-bit cache (odd count), read back
        dict(name="append_prompt_4bit", kind="append", rows=1, tokens=8191, start=37, bits=4, dtype="bfloat16",
             norm=True, keys=True, interleaved=True, max_pos=131072),
        # a few hundred selected rows, and a long cached prefix, for a prompt's next chunk
        dict(name="read_rows", kind="read", n=777, ctx=32768, bits=8, ordered=False),
        dict(name="read_prefix_4bit", kind="read", n=65536, ctx=65536, bits=4, ordered=True),
        # one request's decode step: the selected rows of a long context
        dict(name="sparse_token", kind="sparse", rows=1, heads=16, topk=2048, lo=131072, hi=131072),
        # batched serving of ragged requests
        dict(name="sparse_ragged32", kind="sparse", rows=32, heads=16, topk=2048, lo=1000, hi=16384),
        # a full-attention layer of a few ragged requests
        dict(name="dense_ragged", kind="dense", rows=3, heads=64, lo=777, hi=32768),
        # the same with unsharded heads
        dict(name="dense_128heads", kind="dense", rows=8, heads=128, lo=16001, hi=16384),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(lo * (max(hi, lo) / lo) ** rng.random()))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "rotary", "append", "read", "sparse", "dense"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    size = 4 if dtype == "float32" else 2
    if kind == "norm":
        dim = rng.choice([256, 512, 1536, 2048, 4096, 6144, 7168, 12288, 18432, _log(rng, 64, 8192)])
        return dict(kind=kind, tokens=_log(rng, 1, min(8191, 8191 * 7168 * 2 // (dim * size))), dim=dim, dtype=dtype,
                    residual=rng.random() < 0.6, quant=rng.choice(["none", "none", "128", "128", "row"]),
                    pad=rng.choice([0, 0, 64, 576]))
    if kind == "rotary":
        heads, (nope, rot) = rng.choice([1, 5, 16, 64, 128]), rng.choice([(128, 64), (0, 64), (64, 64), (0, 128), (6, 10)])
        return dict(kind=kind, tokens=_log(rng, 1, min(8191, 4097 * 128 * 128 // (heads * rot * size))), heads=heads,
                    nope=nope, rot=rot, dtype=dtype, interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3,
                    max_pos=rng.choice([4096, 131072, 163840]), yarn=rng.random() < 0.5)
    if kind == "append":
        rows = _log(rng, 1, 64)
        return dict(kind=kind, rows=rows, tokens=1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8191 // rows // (size // 2))),
                    start=_log(rng, 1, 20000), bits=rng.choice([8, 8, 4]), dtype=dtype, norm=rng.random() < 0.7,
                    keys=rng.random() < 0.7, interleaved=rng.random() < 0.5, max_pos=131072)
    if kind == "read":
        ctx = _log(rng, 64, 65536)
        return dict(kind=kind, n=_log(rng, 1, ctx), ctx=ctx, bits=rng.choice([8, 4]), ordered=rng.random() < 0.5)
    rows = _log(rng, 1, 64)
    heads = rng.choice([16, 16, 32, 48, 64, 128])
    if kind == "sparse":
        rows = max(1, rows * 16 // heads)
        hi = _log(rng, 64, min(131072, 524288 // rows))
        return dict(kind=kind, rows=rows, heads=heads, topk=rng.choice([64, 512, 1000, 1024, 2048, 2048]),
                    lo=int(hi * rng.random()), hi=hi)
    hi = _log(rng, 64, min(131072, 16 * 1024 * 1024 // (rows * heads)))
    return dict(kind=kind, rows=rows, heads=heads, lo=int(hi * rng.random()), hi=hi)


def _lens(case: dict) -> list[int]:
    """The requests' lengths: spread over [lo, hi], the longest hi."""
    n, lo, hi = case["rows"], case["lo"], case["hi"]
    u = torch.rand(n, generator=torch.Generator().manual_seed(7000 + n)).tolist()
    u[n // 2] = 1.0
    return [lo + int(round((hi - lo) * x)) for x in u]


# ------------------------------------------------------------ inputs

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


def _rope_angles(case: dict, rot: int, dev) -> tuple[torch.Tensor, float]:
    """Angle per position and pair in float64, and the factor on cos and sin;
    with ``yarn`` stretched 40-fold from 4096 positions (base 10000, 32 and 1
    turns as the ramp's ends)."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=dev)
    freq = 10000.0 ** (-2.0 * i / rot)
    factor = 1.0
    if case.get("yarn"):
        lo, hi = (rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / 40.0 * ramp
        factor = 0.1 * math.log(40.0) + 1.0
    return torch.arange(case["max_pos"], dtype=torch.float64, device=dev)[:, None] * freq, factor


def _rope_table(case: dict, rot: int, dev) -> torch.Tensor:
    """The table a program builds once: [max_pos, rot] float32, cos then sin."""
    a, f = _rope_angles(case, rot, dev)
    return torch.cat([a.cos() * f, a.sin() * f], dim=1).float().contiguous()


def _e4m3_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., 128 or so] float32 -> e4m3 and its scales over the last dim."""
    s = x.abs().amax(-1, keepdim=True).clamp_min(1e-6) / 448.0
    return (x / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s


def _e2m1_codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [n, 512] float32 -> two codes a byte [n, 256] and scale bytes [n, 16]."""
    x = x.reshape(-1, 16, 32)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True).clamp_min(1e-6))  # m in [0.5, 1)
    e = e - 3 + (m > 0.75).to(e.dtype)  # the smallest e with amax <= 6 * 2^e
    a = torch.ldexp(x.abs(), -e)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    code = torch.where(a < 2, 0.0, torch.where(a < 4, 2.0, 4.0)) + (a / step).round()
    code = (code.to(torch.uint8) + 8 * torch.signbit(x).to(torch.uint8)).reshape(-1, 256, 2)
    return code[..., 0] + 16 * code[..., 1], (e + 127).to(torch.uint8).reshape(-1, 16)


def _pack(lat: torch.Tensor, rope: torch.Tensor, bits: int) -> torch.Tensor:
    """Latent rows [n, 656] or [n, 400] of float32 values and bf16 rope."""
    n = lat.shape[0]
    if bits == 8:
        q, s = _e4m3_rows(lat.reshape(n, 4, 128))
        q, s = q.reshape(n, 512).view(torch.uint8), s.reshape(n, 4).contiguous().view(torch.uint8)
    else:
        q, s = _e2m1_codes(lat)
    return torch.cat([q, s, rope.contiguous().view(torch.uint8)], dim=1)


def _values(rows: torch.Tensor) -> torch.Tensor:
    """[n, 576] float32 values of latent rows of either format."""
    n = rows.shape[0]
    if rows.shape[1] == 656:
        q = rows[:, :512].view(torch.float8_e4m3fn).float().reshape(n, 4, 128)
        v = (q * rows[:, 512:528].view(torch.float32)[..., None]).to(torch.bfloat16).float()
        rope = rows[:, 528:]
    else:
        if rows.device not in _CONST:
            _CONST[rows.device] = torch.tensor(E2M1, device=rows.device)
        c = torch.stack([rows[:, :256] & 15, rows[:, :256] >> 4], dim=-1).reshape(n, 16, 32)
        v = _CONST[rows.device][c.int()] * torch.exp2(rows[:, 256:272].float() - 127.0)[..., None]
        rope = rows[:, 272:]
    return torch.cat([v.reshape(n, 512), rope.view(torch.bfloat16).float()], dim=1)


def _pool(g, rows: int, bits: int) -> torch.Tensor:
    """A filled latent pool: rows of differing magnitude."""
    out = []
    for i in range(0, rows, 65536):
        n = min(65536, rows - i)
        out.append(_pack(_randn(g, n, 512) * torch.exp(0.5 * _randn(g, n, 1)), _randn(g, n, 64, dtype=torch.bfloat16), bits))
    return torch.cat(out)


def _pages(case: dict, lens: list[int], seed: int, dev) -> tuple[torch.Tensor, int]:
    """A page table of shuffled physical pages (-1 where a request has none)."""
    need = [-(-n // PAGE) for n in lens]
    total = max(1, sum(need))
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    pt = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        pt[b, :k] = perm[at:at + k]
        at += k
    return pt.to(dev), total


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda:0")
    kind = case["kind"]
    g = torch.Generator(device=dev).manual_seed(1_000_003 * seed + 29)
    dt = DTYPES[case.get("dtype", "bfloat16")]
    if kind == "norm":
        n, d = case["tokens"], case["dim"]
        # `pad`: x is a slice of a wider projection's output
        x = _randn(g, n, d + case["pad"], dtype=dt)[:, :d]
        s = dict(x=x, w=(1 + 0.2 * _randn(g, d)).to(dt), r=None)
        if case["residual"]:
            s["r"] = (3 * _randn(g, n, d)).to(dt)
        return dict(s, kind=kind, quant=case["quant"])
    if kind == "rotary":
        n, h, rot, nope = case["tokens"], case["heads"], case["rot"], case["nope"]
        q = _randn(g, n, h, nope + rot, dtype=dt)
        width = 512 + rot if nope else rot
        return dict(kind=kind, x=q[..., nope:], out=torch.zeros(n, h, width, dtype=dt, device=dev)[..., width - rot:],
                    pos=torch.randint(0, case["max_pos"], (n,), generator=g, device=dev, dtype=torch.int32),
                    table=_rope_table(case, rot, dev), interleaved=case["interleaved"], inverse=case["inverse"])
    if kind == "append":
        B, T = case["rows"], case["tokens"]
        n = B * T
        pt, total = _pages(case, [case["start"] + T] * B, seed, dev)
        bytes_ = 656 if case["bits"] == 8 else 400
        # the latent row is the tail of the fused query-and-latent projection
        s = dict(kind=kind, bits=case["bits"], pt=pt,
                 rows=torch.arange(B, dtype=torch.int32, device=dev).repeat_interleave(T),
                 pos=(torch.arange(T, dtype=torch.int32, device=dev) + case["start"]).repeat(B),
                 latent=_randn(g, n, 1536 + 576, dtype=dt)[:, 1536:], table=_rope_table(case, 64, dev),
                 norm_w=(1 + 0.2 * _randn(g, 512)).to(dt) if case["norm"] else None,
                 pool=torch.zeros(total * PAGE, bytes_, dtype=torch.uint8, device=dev), keys=None, index_k=None,
                 interleaved=case["interleaved"])
        if case["keys"]:
            s["keys"] = _randn(g, n, 128, dtype=dt)
            s["index_k"] = torch.zeros(total, 8448, dtype=torch.uint8, device=dev)
        s["slots"] = (pt[s["rows"].long(), s["pos"].long() // PAGE] * PAGE + s["pos"] % PAGE).to(torch.int32)
        return s
    if kind == "read":
        pool = _pool(g, case["ctx"], case["bits"])
        slots = torch.randperm(case["ctx"], generator=g, device=dev)[:case["n"]]
        return dict(kind=kind, pool=pool, slots=(slots.sort()[0] if case["ordered"] else slots).to(torch.int32))
    lens = _lens(case)
    B, H = case["rows"], case["heads"]
    pt, total = _pages(case, lens, seed, dev)
    s = dict(kind=kind, pool=_pool(g, total * PAGE, 4), q=(2 * _randn(g, B, H, 576)).to(torch.bfloat16),
             out=torch.empty(B, H, 512, dtype=torch.bfloat16, device=dev))
    if kind == "dense":
        return dict(s, pt=pt, lens=torch.tensor(lens, dtype=torch.int32, device=dev), longest=max(lens))
    # a selection: distinct positions ascending as slots, -1 behind a short row's
    K = case["topk"]
    idx = torch.full((B, K), -1, dtype=torch.int32, device=dev)
    for b, n in enumerate(lens):
        p = torch.randperm(n, generator=g, device=dev)[:K].sort()[0]
        idx[b, :len(p)] = pt[b].long()[p // PAGE].mul(PAGE).add(p % PAGE).to(torch.int32)
    return dict(s, idx=idx)


# ------------------------------------------------------------ one pass

def run(s: dict):
    return _run_own(s) if own else _run_plain(s)


def _ops():
    if "ops" not in _CONST:
        import sys
        from pathlib import Path

        path = str(Path(__file__).resolve().parent.parent / "dsa-multi-layer-indexer_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from lagged_indexer_dsa_amd import ops

        _CONST["ops"] = ops
    return _CONST["ops"]


def _run_own(s: dict):
    ops, kind = _ops(), s["kind"]
    if kind == "norm":
        if s["quant"] == "none":
            return ops.rms_norm(s["x"], s["w"], residual=s["r"])
        codes, *rest = ops.rms_norm_quant(s["x"], s["w"], residual=s["r"], group=128 if s["quant"] == "128" else 0)
        return (codes.view(torch.float8_e4m3fn), *rest)
    if kind == "rotary":
        return ops.rotary(s["x"], s["pos"], s["table"], interleaved=s["interleaved"], inverse=s["inverse"], out=s["out"])
    if kind == "append":
        ops.append_tokens(s["pt"], s["rows"], s["pos"], kv_pool=s["pool"], latent=s["latent"], index_k=s["index_k"],
                          keys=s["keys"], cos_sin=s["table"], norm_weight=s["norm_w"], interleaved=s["interleaved"])
        return _caches(s, ops.read_latent_rows(s["pool"], s["slots"]) if s["bits"] == 4 else None)
    if kind == "read":
        return ops.read_latent_rows(s["pool"], s["slots"])
    if "ws" not in s:  # a program allocates its workspace once
        s["ws"] = ops.sparse_mla_workspace(s["q"].shape[0], s["q"].shape[1], 0, s["q"].device)
    if kind == "sparse":
        return ops.sparse_mla_decode(s["q"], s["pool"], s["idx"], workspace=s["ws"], out=s["out"])
    return ops.dense_mla_decode(s["q"], s["pool"], s["pt"], s["lens"], workspace=s["ws"], out=s["out"])


def _caches(s: dict, values):
    """The caches that an append wrote, as the values they hold."""
    out = {}
    if values is None:
        p = s["pool"]
        out = dict(latent=p[:, :512].view(torch.float8_e4m3fn), scale=p[:, 512:528].view(torch.float32),
                   rope=p[:, 528:].view(torch.bfloat16))
    else:
        out = dict(latent=values)
    if s["index_k"] is not None:
        k = s["index_k"]
        out.update(keys=k[:, :8192].view(torch.float8_e4m3fn), key_scale=k[:, 8192:].view(torch.float32))
    return out


def _rotate(x, cos, sin, interleaved):
    """x [..., rot] float32 by cos and sin [..., rot / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _run_plain(s: dict):
    kind = s["kind"]
    if kind == "norm":
        h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s["w"].float()
        n, d = y.shape
        if s["quant"] == "none":
            out = (y.to(s["x"].dtype),)
        else:
            group = 128 if s["quant"] == "128" else d
            y = torch.nn.functional.pad(y, (0, -d % group)).reshape(n, -1, group)
            codes, scale = _e4m3_rows(y)
            out = (codes.reshape(n, -1)[:, :d].contiguous(), scale.reshape(n, -1))
        if s["r"] is not None:
            out += (h.to(s["r"].dtype),)
        return out if len(out) > 1 else out[0]
    if kind == "rotary":
        cos, sin = s["table"][s["pos"].long()][:, None].chunk(2, dim=-1)
        s["out"].copy_(_rotate(s["x"].float(), cos, -sin if s["inverse"] else sin, s["interleaved"]))
        return s["out"]
    if kind == "append":
        slots = (s["pt"][s["rows"].long(), s["pos"].long() // PAGE] * PAGE + s["pos"] % PAGE).long()
        cos, sin = s["table"][s["pos"].long()].chunk(2, dim=-1)
        x = s["latent"].float()
        c = x[:, :512]
        if s["norm_w"] is not None:  # in 64 bits: what lies next to a code's border decides a whole step
            c = c.double()
            c = (c * torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-6) * s["norm_w"].double()).float()
        rope = _rotate(x[:, 512:], cos, sin, s["interleaved"]).to(torch.bfloat16)
        s["pool"][slots] = _pack(c, rope, s["bits"])
        if s["keys"] is not None:
            k = s["keys"].float()
            k = torch.cat([_rotate(k[:, :64], cos, sin, False), k[:, 64:]], dim=1)
            codes, scale = _e4m3_rows(k)
            s["index_k"][:, :8192].view(-1, PAGE, 128)[slots // PAGE, slots % PAGE] = codes.view(torch.uint8)
            s["index_k"].view(torch.float32)[:, 2048:][slots // PAGE, slots % PAGE] = scale[:, 0]
        return _caches(s, _values(s["pool"][slots]).to(torch.bfloat16) if s["bits"] == 4 else None)
    if kind == "read":
        return _values(s["pool"][s["slots"].long()]).to(torch.bfloat16)
    if kind == "sparse":
        slots, ok = s["idx"].long(), s["idx"] >= 0
    else:
        j = torch.arange(s["longest"], device=s["q"].device)
        slots, ok = s["pt"].long()[:, j // PAGE] * PAGE + j % PAGE, j < s["lens"][:, None]
    kv = _values(s["pool"][slots.clamp_min(0).reshape(-1)]).reshape(*slots.shape, 576)
    score = torch.bmm(kv, s["q"].float().transpose(1, 2).contiguous()) * 576 ** -0.5  # [B, keys, H]
    p = torch.softmax(score.masked_fill(~ok[..., None], float("-inf")), dim=1).transpose(1, 2).contiguous()
    o = torch.bmm(p, kv[..., :512].contiguous())
    return torch.where(ok.any(1)[:, None, None], o, 0.0).to(torch.bfloat16)


# ------------------------------------------------------------ what it cannot do without

def work(case: dict) -> dict:
    kind = case["kind"]
    es = 4 if case.get("dtype") == "float32" else 2
    if kind == "norm":
        n, d = case["tokens"], case["dim"]
        row = d * es * (3 if case["residual"] else 1)
        row += d * es if case["quant"] == "none" else d + 4 * (-(-d // 128) if case["quant"] == "128" else 1)
        return dict(bytes=n * row + d * es, flops=n * d * (5 if case["quant"] == "none" else 8))
    if kind == "rotary":
        n, part = case["tokens"], case["heads"] * case["rot"]
        return dict(bytes=n * (2 * part * es + 4 * case["rot"] + 4), flops=n * part * 3)
    if kind == "append":
        n = case["rows"] * case["tokens"]
        row = 576 * es + (656 if case["bits"] == 8 else 400) + 256 + 8 + (128 * es + 132 if case["keys"] else 0)
        row += 400 + 1152 if case["bits"] == 4 else 0
        return dict(bytes=n * row, flops=n * (512 * 8 + 64 * 3 + (128 * 5 if case["keys"] else 0)))
    if kind == "read":
        return dict(bytes=case["n"] * ((656 if case["bits"] == 8 else 400) + 1152 + 4), flops=case["n"] * 512)
    lens, H = _lens(case), case["heads"]
    keys = sum(min(case["topk"], n) for n in lens) if kind == "sparse" else sum(lens)
    return dict(bytes=keys * 400 + case["rows"] * H * 1088 * 2 + (keys * 4 if kind == "sparse" else 0),
                flops=keys * H * 1088 * 2)


# ------------------------------------------------------------ in 64 bits, from the definitions

def _grid(v: torch.Tensor, mantissa: int, emin: int, top: float) -> torch.Tensor:
    """v rounded to the nearest value (ties to even) of a small float format."""
    e = torch.frexp(v)[1].double() - 1
    step = torch.exp2(e.clamp_min(emin) - mantissa)
    return ((v / step).round() * step).clamp(-top, top)


def _exact_rows(c: torch.Tensor, bits: int):
    """Values of the stored groups of c [n, 512] and their scales."""
    n = c.shape[0]
    g = c.reshape(n, 4, 128) if bits == 8 else c.reshape(n, 16, 32)
    top = g.abs().max(-1, keepdim=True)[0].clamp_min(1e-6)
    if bits == 8:
        scale = top / 448
        return _grid(g / scale, 3, -6, 448.0).reshape(n, 512), scale.reshape(n, 4)
    scale = torch.exp2(torch.ceil(torch.log2(top / 6)))
    return (_grid(g / scale, 1, 0, 6.0) * scale).reshape(n, 512), scale


def _exact_turn(x: torch.Tensor, t: torch.Tensor, interleaved: bool, inverse: bool) -> torch.Tensor:
    """x [n, h, rot] as complex numbers times the table's."""
    half = x.shape[-1] // 2
    z = torch.complex(t[:, :half], -t[:, half:] if inverse else t[:, half:])[:, None]
    if interleaved:
        return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:2], half, 2).contiguous()) * z).reshape(x.shape)
    v = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * z
    return torch.cat([v.real, v.imag], dim=-1)


def _decode64(rows: torch.Tensor, bits: int) -> torch.Tensor:
    """[n, 576] of latent rows, read by bit fields; 8-bit values before their
    rounding to bf16."""
    n = rows.shape[0]
    if bits == 8:
        b = rows[:, :512].long()
        e, m = (b >> 3) & 15, b & 7
        v = torch.where(e > 0, (8 + m).double() * torch.exp2(e.double() - 10), m.double() * 2.0 ** -9)
        v = (v * torch.where(b > 127, -1.0, 1.0)).reshape(n, 4, 128)
        v = v * rows[:, 512:528].contiguous().view(torch.float32).double()[..., None]
    else:
        c = torch.empty(n, 512, dtype=torch.long, device=rows.device)
        c[:, 0::2], c[:, 1::2] = (rows[:, :256] % 16).long(), (rows[:, :256] // 16).long()
        e, m = (c >> 1) & 3, c & 1
        v = torch.where(e > 0, (2 + m).double() * torch.exp2(e.double() - 2), m.double() * 0.5)
        v = (v * torch.where(c > 7, -1.0, 1.0)).reshape(n, 16, 32)
        v = torch.ldexp(v, rows[:, 256:272].int()[..., None] - 127)
    rope = rows[:, -128:].contiguous().view(torch.bfloat16).double()
    return torch.cat([v.reshape(n, 512), rope], dim=1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = h + s["r"].double()
        y = h * s["w"].double() / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + 1e-6)
        n, d = y.shape
        if case["quant"] == "none":
            out = [y]
        else:
            group = 128 if case["quant"] == "128" else d
            codes, scales = torch.empty_like(y), []
            for a in range(0, d, group):
                part = y[:, a:a + group]
                scales.append(part.abs().max(1, keepdim=True)[0].clamp_min(1e-6) / 448)
                codes[:, a:a + group] = _grid(part / scales[-1], 3, -6, 448.0)
            out = [codes, torch.cat(scales, dim=1)]
        if s["r"] is not None:
            out.append(h)
        return tuple(out) if len(out) > 1 else out[0]
    if kind == "rotary":
        return _exact_turn(s["x"].double(), s["table"][s["pos"].long()].double(), case["interleaved"], case["inverse"])
    if kind == "append":
        t = s["table"][s["pos"].long()].double()
        x = s["latent"].double()
        c = x[:, :512]
        if s["norm_w"] is not None:
            c = c * s["norm_w"].double() / torch.sqrt((c * c).sum(1, keepdim=True) / 512 + 1e-6)
        turned = _exact_turn(x[:, None, 512:], t, case["interleaved"], False)[:, 0]
        vals, scale = _exact_rows(c, case["bits"])
        slots, n = s["slots"].long(), x.shape[0]
        out = {}
        if case["bits"] == 8:
            rows = s["pool"].shape[0]
            for name, v in (("latent", vals), ("scale", scale), ("rope", turned)):
                out[name] = torch.zeros(rows, v.shape[1], dtype=torch.float64, device=x.device)
                out[name][slots] = v
        else:
            out["latent"] = torch.cat([vals, turned], dim=1)
        if s["keys"] is not None:
            k = s["keys"].double()
            k = torch.cat([_exact_turn(k[:, None, :64], t, False, False)[:, 0], k[:, 64:]], dim=1)
            ks = k.abs().max(1, keepdim=True)[0].clamp_min(1e-6) / 448
            pages = s["index_k"].shape[0]
            out["keys"] = torch.zeros(pages * PAGE, 128, dtype=torch.float64, device=x.device)
            out["key_scale"] = torch.zeros(pages * PAGE, dtype=torch.float64, device=x.device)
            out["keys"][slots], out["key_scale"][slots] = _grid(k / ks, 3, -6, 448.0), ks[:, 0]
            out["keys"], out["key_scale"] = out["keys"].reshape(pages, 8192), out["key_scale"].reshape(pages, PAGE)
        return out
    if kind == "read":
        return _decode64(s["pool"][s["slots"].long()], case["bits"])
    o = torch.zeros(case["rows"], case["heads"], 512, dtype=torch.float64, device=s["q"].device)
    for b in range(case["rows"]):
        if kind == "sparse":
            slots = s["idx"][b][s["idx"][b] >= 0].long()
        else:
            j = torch.arange(int(s["lens"][b]), device=o.device)
            slots = s["pt"][b].long()[j // PAGE] * PAGE + j % PAGE
        if len(slots):
            kv = _decode64(s["pool"][slots], 4)
            e = (s["q"][b].double() @ kv.T) / 24.0
            e = torch.exp(e - e.max(1, keepdim=True)[0])
            o[b] = (e @ kv[:, :512]) / e.sum(1, keepdim=True)
    return o
