"""Performance cases of the operators that take a chunk of new tokens through a layer.

What a program that serves a DSA layer calls when a request brings more than
one token at a time (a part of its prompt, drafted tokens to be verified), and
for the 8-bit products around the attention, each in its plain form (elementary
torch operations in float32) and, with ``own`` set, as the calls of
``lagged_indexer_dsa_amd.ops``:

* ``quant``   -- rows, or rows gated by SiLU, to e4m3 with a scale per 128
  values or per row (``ops.quantize_rows``).
* ``matmul``  -- product of e4m3 rows (a scale per 128 values, or per row) with
  e4m3 weights (a scale per 128 x 128 block) (``ops.fp8_matmul``).
* ``grouped`` -- the same with rows sorted by expert, each expert's weights its
  own, the experts' row counts on the device (``ops.fp8_matmul_grouped``).
* ``scan``    -- indexer scores of the chunks' tokens over the paged index keys,
  -inf behind each token's own position (``ops.chunk_scan``).
* ``attend``  -- attention of the chunks' tokens over the paged latent rows of 8
  or 4 bits, each token up to its own position (``ops.chunk_attention``).

Ranges: 1-8191 rows of 64 to 24576 values, row lengths of products any
multiple of 16, odd numbers of outputs; 1-64 experts, empty ones among them;
1-64 requests with 0-2048 new tokens after 0-131072 cached ones; 16-64 index
heads, 16-128 attention heads.

Latent rows: 656 bytes = 512 e4m3, 4 float32 scales (one per 128 values), 64
bf16; 400 bytes = 512 e2m1 (value 2i in the low half of byte i), 16 e8m0
scales (one per 32 values), 64 bf16.  Index pages: 8448 bytes = 64 keys of 128
e4m3, then their 64 float32 scales.
"""

from __future__ import annotations

import torch

own = False

PAGE = 64
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
_CONST: dict = {}


# ---------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # one token's attention output on its way into the output projection: all latency
        dict(name="quant_token", kind="quant", rows=1, dim=16384, dtype="bfloat16", gate=False, group=128, pad=0),
        # a prompt's MLP activations (odd count), gate and up as the two halves of one projection
        dict(name="quant_gated_prompt", kind="quant", rows=4097, dim=18432, dtype="bfloat16", gate=True, group=128, pad=0),
        # one token through the joint query and latent projection (1536 + 576): weights read once
        dict(name="matmul_token", kind="matmul", rows=1, n=2112, k=7168, row_scale=False, out="bfloat16"),
        # a decode batch's queries out of their latent
        dict(name="matmul_batch", kind="matmul", rows=32, n=24576, k=1536, row_scale=False, out="bfloat16"),
        # a prompt through the MLP's first product (odd count)
        dict(name="matmul_prompt", kind="matmul", rows=4097, n=18432, k=7168, row_scale=False, out="bfloat16"),
        # a decode batch's tokens over many experts, some without a token
        dict(name="grouped_batch", kind="grouped", rows=128, experts=32, n=4096, k=7168, out="bfloat16", extra=0),
        # a prompt's tokens over the same, second product (odd count)
        dict(name="grouped_prompt", kind="grouped", rows=8191, experts=32, n=7168, k=2048, out="bfloat16", extra=0),
        # drafted tokens of a ragged batch
        dict(name="scan_draft", kind="scan", requests=16, tlo=4, thi=4, lo=1000, hi=16384, heads=64, extra=0),
        # a prompt's chunk after a long prefix (odd lengths)
        dict(name="scan_prompt", kind="scan", requests=1, tlo=1023, thi=1023, lo=31751, hi=31751, heads=64, extra=0),
        # drafted tokens of a ragged batch, one tensor-parallel share of heads
        dict(name="attend_draft", kind="attend", requests=16, tlo=4, thi=4, lo=1000, hi=16384, heads=16, bits=8, extra=0),
        # a prompt's chunk after a long prefix (odd lengths)
        dict(name="attend_prompt", kind="attend", requests=1, tlo=1999, thi=1999, lo=16001, hi=16001, heads=16, bits=8,
             extra=0),
        # a batch of chunks and single tokens over the 4-bit cache
        dict(name="attend_mixed_4bit", kind="attend", requests=9, tlo=1, thi=300, lo=0, hi=8192, heads=64, bits=4, extra=3),
    ]


_MATMUL_FLOPS = 2 * 4097 * 18432 * 7168
_ATTEND_PAIRS = 1999 * 16 * 17000  # rows (token and head) times keys
_SCAN_PAIRS = 1023 * 64 * 32262


def _log(rng, lo: int, hi: int) -> int:
    return int(round(lo * (max(hi, lo) / lo) ** rng.random()))


def draw(rng) -> dict:
    kind = rng.choice(["quant", "matmul", "grouped", "scan", "attend", "attend"])
    if kind == "quant":
        dtype, gate = rng.choice(["float32", "bfloat16", "bfloat16", "float16"]), rng.random() < 0.5
        dim = rng.choice([512, 1536, 2048, 6144, 7168, 12288, 16384, 18432, _log(rng, 64, 24576)])
        size = (4 if dtype == "float32" else 2) * (2 if gate else 1) + 1
        return dict(kind=kind, rows=_log(rng, 1, min(8191, 4097 * 18432 * 5 // (dim * size))), dim=dim, dtype=dtype,
                    gate=gate, group=rng.choice([128, 128, 0]), pad=rng.choice([0, 0, 64, 576]))
    out = rng.choice(["bfloat16", "bfloat16", "float32", "float16"])
    if kind == "matmul":
        k = rng.choice([512, 1536, 2048, 6144, 7168, 16384, 16 * _log(rng, 4, 512)])
        n = rng.choice([128, 576, 2112, 6144, 7168, 24576, _log(rng, 64, 8192)])
        return dict(kind=kind, rows=_log(rng, 1, min(8191, _MATMUL_FLOPS // (2 * n * k))), n=n, k=k,
                    row_scale=rng.random() < 0.25, out=out)
    if kind == "grouped":
        k = rng.choice([1536, 2048, 7168, 16 * _log(rng, 4, 448)])
        n = rng.choice([2048, 4096, 7168, _log(rng, 64, 4096)])
        experts = _log(rng, 1, max(1, min(64, 32 * 4096 * 7168 // (n * k))))
        return dict(kind=kind, rows=_log(rng, 1, min(8191, _MATMUL_FLOPS // (2 * n * k))), experts=experts, n=n, k=k,
                    out=out, extra=rng.choice([0, 0, 5]))
    requests = 1 if rng.random() < 0.3 else _log(rng, 2, 64)
    thi = _log(rng, 1, 2048 // requests if rng.random() < 0.5 else 8)
    heads = rng.choice([16, 32, 48, 64, 64] if kind == "scan" else [16, 16, 32, 48, 64, 128])
    pairs = (_SCAN_PAIRS if kind == "scan" else _ATTEND_PAIRS) // (requests * thi * heads)
    hi = max(64, min(_log(rng, 64, 131072), pairs - thi, 2 ** 21 // requests))
    case = dict(kind=kind, requests=requests, tlo=int((thi + 1) * rng.random()), thi=thi, lo=int(hi * rng.random()), hi=hi,
                heads=heads, extra=rng.choice([0, 0, 5]))
    if kind == "attend":
        case["bits"] = rng.choice([8, 8, 4])
    return case


def _spread(n: int, lo: int, hi: int, salt: int) -> list[int]:
    """n numbers over [lo, hi], one of them hi."""
    u = torch.rand(n, generator=torch.Generator().manual_seed(salt + n)).tolist()
    u[n // 2] = 1.0
    return [lo + int(round((hi - lo) * x)) for x in u]


def _chunks(case: dict) -> tuple[list[int], list[int]]:
    """The requests' new tokens, and their cached tokens with those."""
    new = _spread(case["requests"], case["tlo"], case["thi"], 5000)
    old = _spread(case["requests"], case["lo"], case["hi"], 7000)
    return new, [a + b for a, b in zip(new, old)]


def _counts(case: dict) -> list[int]:
    """The experts' rows: uneven, about a quarter of the experts without any."""
    e = case["experts"]
    g = torch.Generator().manual_seed(9000 + e + case["rows"])
    p = torch.exp(torch.randn(e, generator=g)) * (torch.rand(e, generator=g) >= 0.25)
    p[e // 2] += 1.0
    pick = torch.multinomial(p, case["rows"], replacement=True, generator=g)
    return torch.bincount(pick, minlength=e).tolist()


# ------------------------------------------------------------ inputs

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


def _e4m3_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., 128 or so] float32 -> e4m3 and its scales over the last dim."""
    s = x.abs().amax(-1, keepdim=True).clamp_min(1e-6) / 448.0
    return (x / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s


def _groups(x: torch.Tensor, group: int) -> torch.Tensor:
    """x [n, d] as [n, groups, group], zeros behind the last value."""
    group = group or x.shape[1]
    return torch.nn.functional.pad(x, (0, -x.shape[1] % group)).reshape(x.shape[0], -1, group)


def _weights(g, n: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights as a checkpoint holds them: codes that fill the format's range
    and a scale per 128 x 128 block."""
    codes = (_randn(g, n, k) * 100.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, torch.exp(0.3 * _randn(g, -(-n // 128), -(-k // 128))) * 2e-4


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


def _pool(g, rows: int, bits: int) -> torch.Tensor:
    """A filled latent pool: rows of differing magnitude."""
    out = []
    for i in range(0, rows, 65536):
        n = min(65536, rows - i)
        lat, rope = _randn(g, n, 512) * torch.exp(0.5 * _randn(g, n, 1)), _randn(g, n, 64, dtype=torch.bfloat16)
        if bits == 8:
            q, s = _e4m3_rows(lat.reshape(n, 4, 128))
            q, s = q.reshape(n, 512).view(torch.uint8), s.reshape(n, 4).contiguous().view(torch.uint8)
        else:
            q, s = _e2m1_codes(lat)
        out.append(torch.cat([q, s, rope.contiguous().view(torch.uint8)], dim=1))
    return torch.cat(out)


def _pages(lens: list[int], seed: int, dev) -> tuple[torch.Tensor, int]:
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
    g = torch.Generator(device=dev).manual_seed(1_000_003 * seed + 41)
    if kind == "quant":
        n, d, dt = case["rows"], case["dim"], DTYPES[case["dtype"]]
        # `pad`: the rows are slices of a wider projection's output
        x = _randn(g, n, d * (2 if case["gate"] else 1) + case["pad"], dtype=dt)
        return dict(kind=kind, group=case["group"], x=x[:, d:2 * d] if case["gate"] else x[:, :d],
                    gate=x[:, :d] if case["gate"] else None)
    if kind in ("matmul", "grouped"):
        n, k = case["n"], case["k"]
        rows = case["rows"] + case.get("extra", 0)
        a, s = _e4m3_rows(_groups(_randn(g, rows, k) * torch.exp(0.5 * _randn(g, rows, 1)),
                                  0 if case.get("row_scale") else 128))
        state = dict(kind=kind, a=a.reshape(rows, -1)[:, :k].contiguous(), a_scale=s.reshape(rows, -1).contiguous(),
                     dtype=DTYPES[case["out"]])
        if kind == "matmul":
            state["w"], state["w_scale"] = _weights(g, n, k)
            return state
        counts = _counts(case)
        state["w"] = torch.empty(case["experts"], n, k, dtype=torch.float8_e4m3fn, device=dev)
        state["w_scale"] = torch.empty(case["experts"], -(-n // 128), -(-k // 128), device=dev)
        for e in range(case["experts"]):
            state["w"][e], state["w_scale"][e] = _weights(g, n, k)
        ends = [sum(counts[:e]) for e in range(len(counts) + 1)]
        # rows behind the last expert's stay as they are
        return dict(state, ends=ends, offsets=torch.tensor(ends, dtype=torch.int32, device=dev),
                    out=torch.zeros(rows, n, dtype=state["dtype"], device=dev))
    new, lens = _chunks(case)
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    rows = starts[-1] + case["extra"]  # those behind the last request stay as they are
    pt, total = _pages(lens, seed, dev)
    H = case["heads"]
    s = dict(kind=kind, pt=pt, new=new, lens=lens, starts=torch.tensor(starts, dtype=torch.int32, device=dev),
             seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    if kind == "scan":
        q, qs = _e4m3_rows(_randn(g, rows, H, 128))
        k, ks = _e4m3_rows(_randn(g, total * PAGE, 128) * torch.exp(0.3 * _randn(g, total * PAGE, 1)))
        slab = pt.shape[1] * PAGE
        return dict(s, q=q, w=(_randn(g, rows, H) * qs[..., 0] * H ** -0.5).contiguous(),
                    index_k=torch.cat([k.view(torch.uint8).reshape(total, PAGE * 128),
                                       ks.reshape(total, PAGE).contiguous().view(torch.uint8)], dim=1),
                    out=torch.zeros(rows, slab, device=dev))
    return dict(s, q=(2 * _randn(g, rows, H, 576)).to(torch.bfloat16), pool=_pool(g, total * PAGE, case["bits"]),
                out=torch.zeros(rows, H, 512, dtype=torch.bfloat16, device=dev))


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
    if kind == "quant":
        codes, scale = ops.quantize_rows(s["x"], gate=s["gate"], group=s["group"])
        return codes.view(torch.float8_e4m3fn), scale
    if kind == "matmul":
        return ops.fp8_matmul(s["a"], s["a_scale"], s["w"], s["w_scale"], dtype=s["dtype"])
    if kind == "grouped":
        return ops.fp8_matmul_grouped(s["a"], s["a_scale"], s["w"], s["w_scale"], s["offsets"], out=s["out"])
    if kind == "scan":
        return ops.chunk_scan(s["q"], s["w"], s["index_k"], s["pt"], s["starts"], s["seq_lens"], s["out"].shape[1],
                              out=s["out"])
    if "ws" not in s:  # a program allocates its workspace once
        s["ws"] = ops.chunk_workspace(s["q"].shape[0], s["q"].shape[1], s["q"].device)
    return ops.chunk_attention(s["q"], s["pool"], s["pt"], s["starts"], s["seq_lens"], workspace=s["ws"], out=s["out"])


def _values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """[n, k] float32 of e4m3 rows and the scales of their groups (or rows)."""
    k, x = codes.shape[1], codes.float()
    return x * (scale if scale.shape[1] == 1 else scale.repeat_interleave(128, dim=1)[:, :k])


def _weight_values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return _values(codes, scale.repeat_interleave(128, dim=0)[:codes.shape[0]])


def _latent_values(rows: torch.Tensor) -> torch.Tensor:
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


def _requests(s: dict):
    """Per request with new tokens: its number, first row, new and all tokens."""
    at = 0
    for b, (t, n) in enumerate(zip(s["new"], s["lens"])):
        if t:
            yield b, at, t, n
        at += t


def _slots(s: dict, b: int, n: int) -> torch.Tensor:
    """The cache slots of request b's first n tokens."""
    j = torch.arange(n, device=s["pt"].device)
    return s["pt"][b].long()[j // PAGE] * PAGE + j % PAGE


def _run_plain(s: dict):
    kind = s["kind"]
    if kind == "quant":
        x = s["x"].float()
        if s["gate"] is not None:  # in 64 bits: what lies next to a code's border decides a whole step
            gate = s["gate"].double()
            x = (x.double() * gate / (1.0 + torch.exp(-gate))).float()
        codes, scale = _e4m3_rows(_groups(x, s["group"]))
        return codes.reshape(len(x), -1)[:, :x.shape[1]].contiguous(), scale.reshape(len(x), -1)
    if kind == "matmul":
        return (_values(s["a"], s["a_scale"]) @ _weight_values(s["w"], s["w_scale"]).T).to(s["dtype"])
    if kind == "grouped":
        a = _values(s["a"], s["a_scale"])
        for e, (i, j) in enumerate(zip(s["ends"], s["ends"][1:])):
            if j > i:
                s["out"][i:j] = a[i:j] @ _weight_values(s["w"][e], s["w_scale"][e]).T
        return s["out"]
    if kind == "scan":
        H = s["q"].shape[1]
        for b, at, t, n in _requests(s):
            slots = _slots(s, b, n)
            k = s["index_k"][:, :PAGE * 128].view(torch.float8_e4m3fn).reshape(-1, PAGE, 128)
            k = k.view(torch.uint8)[slots // PAGE, slots % PAGE].view(torch.float8_e4m3fn).float()
            ks = s["index_k"].view(torch.float32)[:, PAGE * 32:][slots // PAGE, slots % PAGE]
            own_pos = torch.arange(n - t, n, device=k.device)
            step = max(1, 2 ** 28 // (n * H))
            for i in range(0, t, step):
                m = min(step, t - i)
                q, w = s["q"][at + i:at + i + m].float(), s["w"][at + i:at + i + m]
                score = (torch.relu(q.reshape(m * H, 128) @ k.T).reshape(m, H, n) * w[..., None]).sum(1) * ks
                ahead = torch.arange(n, device=k.device) > own_pos[i:i + m, None]
                s["out"][at + i:at + i + m, :n] = score.masked_fill(ahead, float("-inf"))
            s["out"][at:at + t, n:] = float("-inf")
        return s["out"]
    H = s["q"].shape[1]
    for b, at, t, n in _requests(s):
        kv = _latent_values(s["pool"][_slots(s, b, n)])
        own_pos = torch.arange(n - t, n, device=kv.device)
        step = max(1, 2 ** 28 // (n * H))
        for i in range(0, t, step):
            m = min(step, t - i)
            score = (s["q"][at + i:at + i + m].float().reshape(m * H, 576) @ kv.T).reshape(m, H, n) * 576 ** -0.5
            ahead = torch.arange(n, device=kv.device) > own_pos[i:i + m, None]
            p = torch.softmax(score.masked_fill(ahead[:, None], float("-inf")), dim=-1)
            s["out"][at + i:at + i + m] = (p.reshape(m * H, n) @ kv[:, :512]).reshape(m, H, 512)
    return s["out"]


# ------------------------------------------------------------ what it cannot do without

def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "quant":
        n, d, es = case["rows"], case["dim"], 4 if case["dtype"] == "float32" else 2
        scales = 4 * (-(-d // 128) if case["group"] else 1)
        return dict(bytes=n * (d * es * (2 if case["gate"] else 1) + d + scales), flops=n * d * (7 if case["gate"] else 3))
    if kind in ("matmul", "grouped"):
        m, n, k = case["rows"], case["n"], case["k"]
        used = sum(c > 0 for c in _counts(case)) if kind == "grouped" else 1
        scales = 4 * (m * (1 if case.get("row_scale") else -(-k // 128)) + used * -(-n // 128) * -(-k // 128))
        return dict(bytes=m * k + used * n * k + scales + m * n * (4 if case["out"] == "float32" else 2),
                    flops=2 * m * n * k)
    new, lens = _chunks(case)
    keys = sum(n for t, n in zip(new, lens) if t)
    # a token sees the keys up to its own
    pairs = case["heads"] * sum(t * (n - t) + t * (t + 1) // 2 for t, n in zip(new, lens))
    rows = sum(new)
    if kind == "scan":
        slab = max(1, max(-(-n // PAGE) for n in lens)) * PAGE
        return dict(bytes=keys * 132 + rows * (case["heads"] * 132 + slab * 4), flops=pairs * 2 * 128)
    return dict(bytes=keys * (656 if case["bits"] == 8 else 400) + rows * case["heads"] * 1088 * 2, flops=pairs * 1088 * 2)


# ------------------------------------------------------------ in 64 bits, from the definitions

def _grid(v: torch.Tensor, mantissa: int, emin: int, top: float) -> torch.Tensor:
    """v rounded to the nearest value (ties to even) of a small float format."""
    e = torch.frexp(v)[1].double() - 1
    step = torch.exp2(e.clamp_min(emin) - mantissa)
    return ((v / step).round() * step).clamp(-top, top)


def _e4m3_bits(b: torch.Tensor) -> torch.Tensor:
    """float64 of e4m3 bytes by their fields."""
    b = b.view(torch.uint8).int()
    e, m = (b >> 3) & 15, b & 7
    v = torch.where(e > 0, torch.ldexp((8 + m).double(), e - 10), m.double() * 2.0 ** -9)
    return torch.where(b > 127, -v, v)


def _decode64(rows: torch.Tensor, bits: int) -> torch.Tensor:
    """[n, 576] of latent rows, read by bit fields; a row's value is the
    product of code and scale rounded to bf16 (4 bits: exact as it is)."""
    n = rows.shape[0]
    if bits == 8:
        v = _e4m3_bits(rows[:, :512]).reshape(n, 4, 128) * rows[:, 512:528].contiguous().view(torch.float32).double()[..., None]
        v = _grid(v, 7, -126, float("inf"))
    else:
        c = torch.empty(n, 512, dtype=torch.int32, device=rows.device)
        c[:, 0::2], c[:, 1::2] = (rows[:, :256] % 16).int(), (rows[:, :256] // 16).int()
        e, m = (c >> 1) & 3, c & 1
        v = torch.where(e > 0, (2 + m).double() * torch.exp2(e.double() - 2), m.double() * 0.5)
        v = (v * torch.where(c > 7, -1.0, 1.0)).reshape(n, 16, 32)
        v = torch.ldexp(v, rows[:, 256:272].int()[..., None] - 127)
    rope = rows[:, -128:].contiguous().view(torch.bfloat16).double()
    return torch.cat([v.reshape(n, 512), rope], dim=1)


def _blocks64(codes: torch.Tensor, scale: torch.Tensor, rows: int) -> torch.Tensor:
    """[n, k] of e4m3 codes whose scale [i, j] holds for `rows` rows from i *
    rows and 128 columns from j * 128 (one column of scales: for all)."""
    v = _e4m3_bits(codes)
    width = codes.shape[1] if scale.shape[1] == 1 else 128
    i = torch.arange(codes.shape[0], device=v.device) // rows
    for j in range(scale.shape[1]):
        v[:, j * width:(j + 1) * width] *= scale[i, j].double()[:, None]
    return v


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        y = s["x"].double()
        if case["gate"]:
            y = y * s["gate"].double() * torch.sigmoid(s["gate"].double())
        width = case["group"] or case["dim"]
        codes, scales = torch.empty_like(y), []
        for a in range(0, case["dim"], width):
            part = y[:, a:a + width]
            scales.append(part.abs().max(1, keepdim=True)[0].clamp_min(1e-6) / 448)
            codes[:, a:a + width] = _grid(part / scales[-1], 3, -6, 448.0)
        return codes, torch.cat(scales, dim=1)
    if kind == "matmul":
        return _blocks64(s["a"], s["a_scale"], 1) @ _blocks64(s["w"], s["w_scale"], 128).T
    if kind == "grouped":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
        for e, n in enumerate(_counts(case)):
            i = s["ends"][e]
            if n:
                a = _blocks64(s["a"][i:i + n], s["a_scale"][i:i + n], 1)
                out[i:i + n] = a @ _blocks64(s["w"][e], s["w_scale"][e], 128).T
        return out
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    new, lens = _chunks(case)
    for b, (t, n) in enumerate(zip(new, lens)):
        i0 = sum(new[:b])
        where = torch.arange(n, device=out.device)
        slots = s["pt"][b].long()[where // PAGE] * PAGE + where % PAGE
        if kind == "scan":
            page = s["index_k"][slots // PAGE]
            at = (slots % PAGE)[:, None]
            k = _e4m3_bits(page.gather(1, at * 128 + torch.arange(128, device=out.device)))
            ks = page[:, PAGE * 128:].contiguous().view(torch.float32).gather(1, at)[:, 0].double()
        else:
            kv = _decode64(s["pool"][slots], case["bits"])
        for i in range(t):
            seen = n - t + i + 1
            if kind == "scan":
                hits = (_e4m3_bits(s["q"][i0 + i]) @ k[:seen].T).clamp_min(0.0)
                out[i0 + i, :seen] = (s["w"][i0 + i].double() @ hits) * ks[:seen]
                out[i0 + i, seen:] = float("-inf")
            else:
                e = (s["q"][i0 + i].double() @ kv[:seen].T) / 24.0
                e = torch.exp(e - e.max(1, keepdim=True)[0])
                out[i0 + i] = (e @ kv[:seen, :512]) / e.sum(1, keepdim=True)
    return out
