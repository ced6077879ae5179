"""Cache operators: attention over a shared prefix and own caches, attention
weight per key, eviction -- each against its definition in 64 bits.

Tolerances (u = half a unit of the inputs' type relative to the value, 2^-8 for
bf16 and 2^-11 for fp16):

* attention output: P is rounded once for the tensor core (u * sum p|v|) and the
  result once (u * |o|); the scores' fp32 error ds, the sums and exp2 add
  (2 ds + 2^-18) * sum p|v|; fp16 P below 2^-14 is off by up to 2^-25 absolute,
  relative to a maximum of 1 in its own range: 2^-25 * keys * max|v|;
* ds: a dot product of D products summed in fp32, then scaled: an element's
  error is at most (D + 4) 2^-23 of scale * sum |q||k| (the tensor core may
  truncate, hence a whole unit per addition);
* lse: ds + 2^-20 (1 + |lse|) (exp2, log2 and the sums);
* weights: every term relative 2 ds + 2^-18, or ds + the given lse's own
  rounding 2^-24 |lse| with it.
"""

from __future__ import annotations

import math

import pytest
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


# ---------------------------------------------------------------------------
# Definitions in 64 bits
# ---------------------------------------------------------------------------


def rows_of(q, kp, k, lens, plens, b, head, scale, causal):
    """(scores [S_q, keys] with -inf where hidden, error of a score, key count of the prefix)."""
    B, Hq, Sq, D = q.shape
    parts, hidden = [], []
    P = 0
    if kp is not None:
        G, Hkv = kp.shape[:2]
        g = b // (B // G)
        P = kp.shape[2] if plens is None else min(max(plens[g], 0), kp.shape[2])
        parts.append(kp[g, head // (Hq // Hkv), :P].double())
        hidden.append(torch.zeros(Sq, P, dtype=torch.bool, device=q.device))
    if k is not None:
        Hkv, C = k.shape[1:3]
        n = C if lens is None else min(max(lens[b], 0), C)
        parts.append(k[b, head // (Hq // Hkv), :n].double())
        j = torch.arange(n, device=q.device)
        r = torch.arange(Sq, device=q.device)[:, None]
        hidden.append(j > n - Sq + r if causal else torch.zeros(Sq, n, dtype=torch.bool,
                                                                device=q.device))
    keys = torch.cat(parts)
    qd = q[b, head].double()
    s = (qd @ keys.T * scale).masked_fill(torch.cat(hidden, 1), -math.inf)
    mag = (qd.abs() @ keys.abs().T).max().item() * abs(scale) if keys.shape[0] else 0.0
    return s, (D + 4) * 2.0**-23 * mag, P


def ref_attention(q, kp, vp, k, v, lens=None, plens=None, scale=None, causal=True):
    B, Hq, Sq, D = q.shape
    scale = D**-0.5 if scale is None else scale
    u = U[q.dtype]
    out = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64, device=q.device)
    ltol = torch.zeros_like(lse)
    for b in range(B):
        for h in range(Hq):
            s, ds, P = rows_of(q, kp, k, lens, plens, b, h, scale, causal)
            if s.shape[1] == 0:
                continue
            vals = []
            if kp is not None:
                g = b // (B // kp.shape[0])
                vals.append(vp[g, h // (Hq // kp.shape[1]), :P].double())
            if k is not None:
                vals.append(v[b, h // (Hq // k.shape[1]), :s.shape[1] - P].double())
            vals = torch.cat(vals)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z.masked_fill(z.isinf(), 0)[:, None])
            out[b, h] = p @ vals
            pv = p @ vals.abs()
            tol[b, h] = (u + 2 * ds + 2.0**-18) * pv + u * out[b, h].abs() + 1e-7
            if q.dtype == torch.float16:
                tol[b, h] += 2.0**-25 * s.shape[1] * vals.abs().max() + 2.0**-25
            lse[b, h] = z
            ltol[b, h] = ds + 2.0**-20 * (1 + z.abs().masked_fill(z.isinf(), 0))
    return out, tol, lse, ltol


def ref_weights(q, k, w, lens=None, lse=None, scale=None, causal=True):
    B, Hq, Sq, D = q.shape
    Hkv, C = k.shape[1:3]
    scale = D**-0.5 if scale is None else scale
    acc = torch.zeros(B, Hkv, C, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(acc)
    for b in range(B):
        for h in range(Hq):
            s, ds, _ = rows_of(q, None, k, lens, None, b, h, scale, causal)
            z = torch.logsumexp(s, 1) if lse is None else lse[b, h].double()
            rel = 2 * ds + 2.0**-18
            if lse is not None:
                rel += 2.0**-24 * z[~z.isinf()].abs().max().item() if (~z.isinf()).any() else 0
            dead = z == -math.inf
            p = torch.exp(s - z.masked_fill(dead, 0)[:, None]).masked_fill(dead[:, None], 0)
            acc[b, h // (Hq // Hkv), :s.shape[1]] += p.sum(0)
            tol[b, h // (Hq // Hkv), :s.shape[1]] += rel * p.sum(0)
    if w is not None:
        acc += w.double()
    return acc, tol + 2.0**-22 * acc.abs() + 1e-30


def ref_evict(w, keep, lens, sink, recent):
    """Index lists [B][H] by a plain sort of (weight, -index)."""
    B, H, C = w.shape
    out = []
    for b in range(B):
        n = C if lens is None else min(max(lens[b], 0), C)
        row = []
        for h in range(H):
            key = []
            for j, x in enumerate(w[b, h, :n].tolist()):
                forced = j < sink or j >= n - recent
                rank = 2 if forced else (0 if math.isnan(x) else 1)
                key.append((-rank, 0.0 if forced or math.isnan(x) else -x, j))
            row.append(sorted(j for _, _, j in sorted(key)[:keep]))
        out.append(row)
    return out


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def cache(g, B, H, S, D, dtype, layout="bhsd"):
    shape = (B, S, H, D) if layout == "bshd" else (B, H, S, D)
    x = torch.randn(shape, generator=g).to(dtype).cuda()
    return x.transpose(1, 2) if layout == "bshd" else x


def poison(x, lens):
    """NaN and infinities in the rows past each length."""
    for b, n in enumerate(lens):
        n = min(max(n, 0), x.shape[2])
        x[b, :, n:] = float("nan")
        x[b, :, n + 1::2] = float("inf")


def make(case, seed=0):
    B, Hq, Hkv, Sq, G, P, C, D, dtype, layout = case
    g = torch.Generator().manual_seed(seed)
    q = cache(g, B, Hq, Sq, D, dtype, "bshd")
    kp, vp = (cache(g, G, Hkv, P, D, dtype, layout) for _ in range(2)) if P else (None, None)
    k, v = (cache(g, B, Hkv, C, D, dtype, layout) for _ in range(2)) if C else (None, None)
    return q, kp, vp, k, v


BF, FP = torch.bfloat16, torch.float16
#        B Hq Hkv Sq G  P     C    D   type layout
ATTENTION = [
    (1, 1, 1, 1, 1, 0, 1, 64, BF, "bhsd"),          # one key
    (1, 2, 1, 1, 1, 1, 1, 8, FP, "bhsd"),           # one prefix key, one own key
    (4, 4, 4, 1, 1, 300, 70, 96, BF, "bhsd"),       # decode, one head per key/value head
    (3, 8, 2, 1, 1, 1000, 33, 128, FP, "bshd"),     # grouped heads, token-major caches
    (6, 14, 2, 1, 3, 129, 65, 80, BF, "bshd"),      # seven heads a group, three prefixes
    (5, 8, 1, 4, 1, 255, 90, 64, FP, "bhsd"),       # drafts: 32 rows a cache
    (2, 4, 2, 17, 2, 513, 40, 72, BF, "bhsd"),      # 34 rows: past a row tile
    (2, 4, 1, 70, 1, 700, 100, 128, BF, "bhsd"),    # questions: hundreds of rows
    (3, 2, 2, 130, 1, 64, 130, 96, FP, "bshd"),     # every token new
    (40, 4, 1, 1, 1, 777, 20, 128, BF, "bhsd"),     # 160 rows share a prefix
    (2, 2, 2, 3, 1, 0, 2000, 33, BF, "bhsd"),       # a head dim without 16-byte rows
    (2, 4, 2, 1, 1, 0, 5000, 120, FP, "bhsd"),      # no prefix, several ranges
    (4, 4, 2, 2, 2, 600, 0, 40, BF, "bhsd"),        # no own cache
    (1, 8, 8, 200, 1, 0, 333, 64, BF, "bhsd"),      # a chunk of a prompt
    (2, 16, 2, 64, 1, 1500, 64, 128, FP, "bhsd"),   # 512 rows a cache
    (8, 32, 8, 9, 1, 0, 1500, 96, BF, "bshd"),      # several key blocks an item
    (40, 8, 8, 1, 1, 5000, 30, 128, BF, "bhsd"),
    (16, 16, 16, 40, 1, 0, 1200, 64, FP, "bhsd"),   # whole caches an item
    (16, 16, 16, 33, 1, 700, 500, 128, BF, "bhsd"),
    (6, 4, 2, 33, 2, 300, 80, 96, FP, "bhsd"),      # one walk over a shared prefix and own keys
]


def ids(c):
    return "-".join(str(x).replace("torch.", "") for x in c)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", ATTENTION, ids=ids)
def test_attention_matches_definition(cuda, case, causal):
    from minference import ops

    q, kp, vp, k, v = make(case)
    out, lse = ops.shared_prefix_attention(q, kp, vp, k, v, causal=causal, return_lse=True)
    ref, tol, rl, lt = ref_attention(q, kp, vp, k, v, causal=causal)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    assert ((out.double() - ref).abs() <= tol).all(), ((out.double() - ref).abs() / tol).max()
    assert torch.equal(lse.isinf(), rl.isinf())
    seen = ~rl.isinf()
    assert ((lse.double() - rl).abs() <= lt)[seen].all()
    assert (out[~seen] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTENTION, ids=ids)
def test_attention_ragged_lengths_and_stale_rows(cuda, case):
    """Lengths of zero and one, past the capacity and below the new tokens;
    whatever lies behind them stays out."""
    from minference import ops

    q, kp, vp, k, v = make(case, 1)
    B, Hq, Hkv, Sq, G, P, C, D, dtype, layout = case
    lens = [[C, 0, 1, Sq, C + 5, max(0, Sq - 1), -3, C // 2][b % 8] for b in range(B)]
    plens = [[P // 2, P, 0][g % 3] for g in range(G)]
    kw = {}
    if P:
        kw["prefix_lengths"] = torch.tensor(plens, dtype=torch.int32).cuda()
        poison(kp, plens), poison(vp, plens)
    lt = None
    if C:
        lt = torch.tensor(lens, dtype=torch.int64).cuda()
        poison(k, lens), poison(v, lens)
    out, lse = ops.shared_prefix_attention(q, kp, vp, k, v, lt, return_lse=True, **kw)
    ref, tol, rl, ltol = ref_attention(q, kp, vp, k, v, lens, plens)
    assert ((out.double() - ref).abs() <= tol).all()
    assert torch.equal(lse.isinf(), rl.isinf())
    seen = ~rl.isinf()
    assert ((lse.double() - rl).abs() <= ltol)[seen].all()
    assert (out[~seen] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.7, 3.0])
def test_attention_scales(cuda, scale):
    from minference import ops

    for case in (ATTENTION[3], ATTENTION[7], ATTENTION[9]):
        q, kp, vp, k, v = make(case, 2)
        out = ops.shared_prefix_attention(q, kp, vp, k, v, scale=scale)
        ref, tol, _, _ = ref_attention(q, kp, vp, k, v, scale=scale)
        assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 70, 200])
def test_a_scale_that_is_nan_gives_nan(cuda, Sq):
    from minference import ops

    q, kp, vp, k, v = make((2, 4, 2, Sq, 1, 300, 250, 64, BF, "bhsd"), 39)
    out, lse = ops.shared_prefix_attention(q, kp, vp, k, v, scale=math.nan, return_lse=True)
    assert out.isnan().all() and lse.isnan().all()
    assert ops.accumulate_attention_weights(q, k, scale=math.nan).isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Sq", [1, 5, 70])
def test_attention_rising_scores(cuda, Sq, dtype):
    """Every block's scores lie above those before, by hundreds in all: the
    running reference has to move, at every height of the row tile."""
    from minference import ops

    q, kp, vp, k, v = make((2, 8, 2, Sq, 1, 900, 200, 128, dtype, "bhsd"), 30)
    ramp = torch.linspace(0.2, 12.0, 1100, device="cuda")
    q = q.abs()
    kp = (kp.abs() * ramp[:900, None]).to(dtype)
    k = (k.abs() * ramp[900:, None]).to(dtype)
    out, lse = ops.shared_prefix_attention(q, kp, vp, k, v, return_lse=True)
    ref, tol, rl, lt = ref_attention(q, kp, vp, k, v)
    assert rl.max() - (q[0, 0, 0].double() @ kp[0, 0, 0].double()) * 128**-0.5 > 60
    assert ((out.double() - ref).abs() <= tol).all()
    assert ((lse.double() - rl).abs() <= lt).all()
    # and falling: what comes first stays the reference
    out = ops.shared_prefix_attention(q, kp.flip(2), vp.flip(2), k, v)
    ref, tol, _, _ = ref_attention(q, kp.flip(2), vp.flip(2), k, v)
    assert ((out.double() - ref).abs() <= tol).all()


def blocks_an_item(q, kp, k):
    """64-key blocks that a tile walks in one item, at least: from the partial
    results a row has (0 bytes: one), where one kind of item covers the call."""
    from minference import _native

    B, Hq, Sq, D = q.shape
    Hkv, C = k.shape[1:3]
    G, P = (kp.shape[0], kp.shape[2]) if kp is not None else (1, 0)
    none = (0, 0, 0, 0)
    need = _native.lib().mi_shared_prefix_fwd_workspace_size(_native.SHARED_PREFIX_ARGS.pack(
        *none * 6, 0, 0, 0, B, Hq, Hkv, Sq, G, P, C, D, 1, 1, 1.0))
    slots = max(1, round(need / (B * Hq * Sq * (4 * D + 8))))
    return (-(-P // 64) + -(-C // 64)) / slots


#   B  Hq  Hkv Sq   P    C     D   lengths / prefix lengths
MIXED = [
    (4, 32, 8, 100, 0, 1500, 128, [860, 1500, 99, 70], None),  # rows wrap into the next head
    (1, 4, 2, 1000, 0, 1000, 64, None, None),         # ranges that start among the new tokens
    (2, 4, 2, 200, 0, 300, 96, [150, 300], None),     # fewer keys than new tokens
    (16, 16, 8, 100, 256, 600, 128, [600, 90, 80, 555] * 4, [256, 0]),  # one walk over both
    (16, 16, 16, 40, 0, 1200, 64, None, None),        # every row of a warp sees something
]


@pytest.mark.gpu
@pytest.mark.parametrize("rise", [3, 13, 100])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("case", MIXED, ids=ids)
def test_attention_rising_scores_beside_rows_that_see_nothing(cuda, case, dtype, rise):
    """Scores rise by `rise` from each 64-key block to the next: a row's reference
    has to move from one block of an item to a later one, also while other rows
    of its warp have none yet."""
    from minference import ops

    B, Hq, Hkv, Sq, P, C, D, lens, plens = case
    G = 2 if P else 1
    q, kp, vp, k, v = make((B, Hq, Hkv, Sq, G, P, C, D, dtype, "bhsd"), 33)
    assert blocks_an_item(q, kp, k) > 1
    q = (0.25 * q).contiguous()
    q[..., 0] = 4
    step = torch.arange((P + C + 63) // 64, device="cuda").repeat_interleave(64)
    step = (step * (rise * D**0.5 / 4)).to(dtype)
    k[..., 0] = step[P:P + C]
    if P:
        kp[..., 0] = step[:P]
    cu = [None if x is None else torch.tensor(x, dtype=torch.int32).cuda() for x in (lens, plens)]
    out, lse = ops.shared_prefix_attention(q, kp, vp, k, v, cu[0], prefix_lengths=cu[1],
                                           return_lse=True)
    ref, tol, rl, lt = ref_attention(q, kp, vp, k, v, lens, plens)
    assert torch.equal(lse.isinf(), rl.isinf())
    seen = ~rl.isinf()
    assert ((lse.double() - rl).abs() <= lt)[seen].all()
    assert ((out.double() - ref).abs() <= tol).all()
    assert (out[~seen] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [96, 40, 33])
def test_attention_writes_the_given_view_only(cuda, D):
    from minference import ops

    case = (3, 4, 2, 2, 1, 200, 50, D, BF, "bhsd")
    q, kp, vp, k, v = make(case, 3)
    pitch = -(-D // 8) * 8 + 8
    buf = torch.full((3, 2, 6, pitch), 7.0, dtype=BF, device="cuda")
    view = buf.transpose(1, 2)[:, 1:5, :, :D]
    res = ops.shared_prefix_attention(q, kp, vp, k, v, out=view)
    assert res.data_ptr() == view.data_ptr()
    ref, tol, _, _ = ref_attention(q, kp, vp, k, v)
    assert ((view.double() - ref).abs() <= tol).all()
    assert (buf[:, :, 0] == 7).all() and (buf[:, :, 5] == 7).all() and (buf[..., D:] == 7).all()


@pytest.mark.gpu
def test_attention_unaligned_and_expanded_inputs(cuda):
    """Views that 16-byte loads cannot read, one cache expanded over the batch."""
    from minference import ops

    g = torch.Generator().manual_seed(4)
    base = torch.randn(2, 2, 300, 66, generator=g).to(FP).cuda()
    kp, vp = base[:1, :, :, 1:65], base[1:, :, :, 2:66]
    q = torch.randn(3, 4, 1, 65, generator=g).to(FP).cuda()[..., 1:]
    k = torch.randn(1, 2, 40, 64, generator=g).to(FP).cuda().expand(3, -1, -1, -1)
    v = torch.randn(3, 2, 40, 64, generator=g).to(FP).cuda()
    out = ops.shared_prefix_attention(q, kp, vp, k, v)
    ref, tol, _, _ = ref_attention(q, kp, vp, k, v)
    assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_attention_key_offsets_past_32_bits(cuda):
    """A token-major cache whose last rows lie past 2^31 elements."""
    from minference import ops

    S, H, D = 70000, 256, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.empty(1, S, H, D, dtype=BF, device="cuda").normal_(generator=g).transpose(1, 2)
    v = torch.empty(1, S, H, D, dtype=BF, device="cuda").normal_(generator=g).transpose(1, 2)
    assert (S - 1) * H * D > 2**31
    q = torch.empty(1, 2, 1, D, dtype=BF, device="cuda").normal_(generator=g)
    for a, b in ((k, v), ):
        out = ops.shared_prefix_attention(q, None, None, a[:, -2:], b[:, -2:])
        ref, tol, _, _ = ref_attention(q, None, None, a[:, -2:], b[:, -2:])
        assert ((out.double() - ref).abs() <= tol).all()
    q = torch.empty(128, 2, 1, D, dtype=BF, device="cuda").normal_(generator=g)
    out = ops.shared_prefix_attention(q, k[:, -2:], v[:, -2:], None, None)
    ref, tol, _, _ = ref_attention(q[:2], k[:, -2:], v[:, -2:], None, None)
    assert ((out[:2].double() - ref).abs() <= tol).all()
    w = ops.accumulate_attention_weights(q[:1], k[:, -2:])
    wr, wt = ref_weights(q[:1], k[:, -2:], None)
    assert ((w.double() - wr).abs() <= wt).all()


# ---------------------------------------------------------------------------
# Weights
# ---------------------------------------------------------------------------

#        B Hq Hkv Sq  C    D  type layout
WEIGHTS = [
    (1, 1, 1, 1, 1, 64, BF, "bhsd"),
    (3, 8, 2, 1, 500, 128, FP, "bshd"),
    (2, 7, 1, 1, 3000, 80, BF, "bhsd"),
    (2, 4, 4, 5, 100, 96, BF, "bhsd"),
    (1, 2, 2, 64, 1000, 96, FP, "bhsd"),      # a prompt's last queries
    (2, 4, 2, 70, 70, 40, BF, "bshd"),
    (1, 4, 2, 257, 257, 128, BF, "bhsd"),     # every query
    (1, 3, 1, 300, 777, 64, FP, "bhsd"),
    (1, 2, 1, 9, 65, 33, BF, "bhsd"),
    (2, 2, 2, 129, 513, 72, FP, "bshd"),
    (6, 32, 32, 12, 2000, 64, BF, "bhsd"),    # several key tiles an item
    (1, 16, 16, 1500, 1500, 128, FP, "bhsd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("case", WEIGHTS, ids=ids)
def test_weights_match_definition(cuda, case, given, causal):
    from minference import ops

    B, Hq, Hkv, Sq, C, D, dtype, layout = case
    q, _, _, k, v = make((B, Hq, Hkv, Sq, 1, 0, C, D, dtype, layout), 6)
    lse = ref_attention(q, None, None, k, v, causal=causal)[2].float() if given else None
    w = ops.accumulate_attention_weights(q, k, lse=lse, causal=causal)
    ref, tol = ref_weights(q, k, None, lse=lse, causal=causal)
    assert w.dtype == torch.float32 and ((w.double() - ref).abs() <= tol).all()
    # every row that sees something gives away exactly its probability
    if not given and (Sq <= C or not causal):
        total = w.double().sum((1, 2))
        assert torch.allclose(total, torch.full_like(total, Hq * Sq), rtol=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("case", WEIGHTS, ids=ids)
def test_weights_ragged_and_added_in_place(cuda, case, given):
    from minference import ops

    B, Hq, Hkv, Sq, C, D, dtype, layout = case
    q, _, _, k, v = make((B, Hq, Hkv, Sq, 1, 0, C, D, dtype, layout), 7)
    for lens in ([C // 2, C, 0], [0, 1, C], [min(Sq, C) - 1, C - 1, C + 9]):
        lens = (lens * B)[:B]
        kk = k.clone()
        poison(kk, lens)
        lt = torch.tensor(lens, dtype=torch.int32).cuda()
        lse = ref_attention(q, None, None, kk, v, lens)[2].float() if given else None
        big = torch.rand(B, Hkv, C + 3, device="cuda")
        w0, w = big.clone(), big[:, :, 1:C + 1]
        got = ops.accumulate_attention_weights(q, kk, w, lt, lse=lse)
        assert got.data_ptr() == w.data_ptr()
        ref, tol = ref_weights(q, kk, w0[:, :, 1:C + 1], lens, lse=lse)
        assert ((w.double() - ref).abs() <= tol).all()
        for b, n in enumerate(lens):
            n = min(max(n, 0), C)
            assert torch.equal(big[b, :, 1 + n:], w0[b, :, 1 + n:])
        assert torch.equal(big[:, :, 0], w0[:, :, 0])
        out = torch.full((B, Hkv, C), 5.0, device="cuda")
        ops.accumulate_attention_weights(q, kk, w0[:, :, 1:C + 1], lt, lse=lse, out=out)
        assert torch.equal(out, w)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 64, 200])
@pytest.mark.parametrize("scale", [0.0, -0.7, 3.0])
def test_weights_scales(cuda, Sq, scale):
    from minference import ops

    q, _, _, k, _ = make((2, 4, 2, Sq, 1, 0, 777, 96, FP, "bhsd"), 31)
    w = ops.accumulate_attention_weights(q, k, scale=scale)
    ref, tol = ref_weights(q, k, None, scale=scale)
    assert ((w.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 64, 300])
def test_weights_rising_scores(cuda, Sq):
    from minference import ops

    for flip in (False, True):
        q, _, _, k, _ = make((1, 4, 2, Sq, 1, 0, 1300, 128, BF, "bhsd"), 32)
        q = q.abs()
        ramp = torch.linspace(0.2, 12.0, 1300, device="cuda")
        k = (k.abs() * (ramp.flip(0) if flip else ramp)[:, None]).to(BF)
        w = ops.accumulate_attention_weights(q, k)
        ref, tol = ref_weights(q, k, None)
        assert ((w.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 5, 20, 33, 40, 70, 300])
def test_weights_of_nothing_are_exactly_zero(cuda, Sq):
    """Rows whose lse is -inf add nothing, and probabilities far below fp32's range
    are 0, whatever path a key takes: eviction's ties among zeros depend on it."""
    from minference import ops

    q, _, _, k, _ = make((2, 4, 2, Sq, 1, 0, 900, 96, BF, "bhsd"), 34)
    none = torch.full((2, 4, Sq), -math.inf, device="cuda")
    for causal in (False, True):
        assert (ops.accumulate_attention_weights(q, k, lse=none, causal=causal) == 0).all()
    some = ref_attention(q, None, None, k, k, causal=False)[2].float()
    some[:, :, ::2] = -math.inf
    w = ops.accumulate_attention_weights(q, k, lse=some, causal=False)
    ref, tol = ref_weights(q, k, None, lse=some, causal=False)
    assert ((w.double() - ref).abs() <= tol).all()
    q = (0.25 * q).contiguous()
    q[..., 0] = 4
    far = torch.zeros(900, dtype=torch.bool, device="cuda")
    far[100:700] = True
    k[..., 0] = torch.where(far, -1000.0, 0.0).to(BF)  # 400 below the others
    lse = ref_attention(q, None, None, k, k, causal=False)[2].float()
    for z in (None, lse):
        w = ops.accumulate_attention_weights(q, k, lse=z, causal=False)
        assert (w[..., far] == 0).all() and (w[..., ~far] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [5, 20, 40, 300])
def test_weights_of_an_lse_far_too_small_overflow(cuda, Sq):
    """A sum of exponentials past fp32's range is infinite, in every column."""
    from minference import ops

    q, _, _, k, _ = make((1, 2, 2, Sq, 1, 0, 300, 64, BF, "bhsd"), 35)
    lse = torch.full((1, 2, Sq), -500.0, device="cuda")
    assert (ops.accumulate_attention_weights(q, k, lse=lse, causal=False) == math.inf).all()
    for at in range(8):  # one such row among rows that add nothing
        lse = torch.full((1, 2, Sq), -math.inf, device="cuda")
        lse[:, :, at % Sq] = -500.0
        assert (ops.accumulate_attention_weights(q, k, lse=lse, causal=False) == math.inf).all()


@pytest.mark.gpu
def test_weights_of_an_attention_with_prefix(cuda):
    """lse of the attention: own weights plus the prefix's add up to the rows."""
    from minference import ops

    for Sq, P, C in ((1, 400, 90), (96, 300, 150)):
        q, kp, vp, k, v = make((2, 8, 2, Sq, 1, P, C, 128, BF, "bhsd"), 8)
        _, lse = ops.shared_prefix_attention(q, kp, vp, k, v, return_lse=True)
        w = ops.accumulate_attention_weights(q, k, lse=lse)
        flat = q.transpose(0, 1).reshape(1, 2, 4, 2, Sq, 128).transpose(2, 3)
        # the prefix as a cache of its own that every sequence's rows see in full
        wp = ops.accumulate_attention_weights(q, kp.expand(2, -1, -1, -1), lse=lse, causal=False)
        assert flat.numel() == q.numel()
        total = w.double().sum((1, 2)) + wp.double().sum((1, 2))
        assert torch.allclose(total, torch.full_like(total, 8 * Sq), rtol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Sq, P, C", [(1, 0, 700), (1, 900, 50), (3, 40, 0), (4, 0, 4000),
                                      (40, 0, 900), (70, 700, 100), (130, 0, 333)])
def test_nan_queries_come_out_as_nan(cuda, Sq, P, C, dtype):
    """A NaN in a query is no row that sees nothing: its output and log-sum-exp are
    NaN, the keys it sees get NaN weights, and no other row or head changes."""
    from minference import ops

    q, kp, vp, k, v = make((3, 4, 2, Sq, 1, P, C, 128, dtype, "bhsd"), 36)
    lens = [C, C // 2, 0]
    lt = torch.tensor(lens, dtype=torch.int32).cuda() if C else None
    bad = torch.zeros(3, 4, Sq, dtype=torch.bool, device="cuda")
    bad[0, 1, Sq // 2] = bad[1, 0, Sq - 1] = bad[2, 0, 0] = True
    q2 = torch.where(bad[..., None] & (torch.arange(128, device="cuda") == 5), float("nan"), q)
    o, z = ops.shared_prefix_attention(q, kp, vp, k, v, lt, return_lse=True)
    o2, z2 = ops.shared_prefix_attention(q2, kp, vp, k, v, lt, return_lse=True)
    nan = bad & ~z.isinf()
    assert nan.any()
    assert o2[nan].isnan().all() and z2[nan].isnan().all()
    assert torch.equal(o2[~nan], o[~nan]) and torch.equal(z2[~nan], z[~nan])
    if not C:
        return
    seen = torch.zeros(3, 2, C, dtype=torch.bool, device="cuda")
    for b, h, r in bad.nonzero().tolist():
        seen[b, h // 2, :max(0, lens[b] - (Sq - 1 - r))] = True
    for lse, lse2 in ((None, None), (z, z2)):
        w = ops.accumulate_attention_weights(q, k, None, lt, lse=lse)
        w2 = ops.accumulate_attention_weights(q2, k, None, lt, lse=lse2)
        assert torch.equal(w2.isnan(), seen)
        assert torch.equal(w2[~seen], w[~seen])


# ---------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------


def check_evicted(res, k, v, w, keep, lens, sink, recent):
    B, H, C = w.shape
    ref = ref_evict(w, keep, lens, sink, recent)
    n = [min(keep, C if lens is None else min(max(lens[b], 0), C)) for b in range(B)]
    assert res.lengths.tolist() == n
    idx = torch.full((B, H, keep), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(H):
            idx[b, h, :n[b]] = torch.tensor(ref[b][h], dtype=torch.int32)
    assert torch.equal(res.index.cpu(), idx)
    for b in range(B):
        for h in range(H):
            at = idx[b, h, :n[b]].long().cuda()
            for got, src in ((res.k, k), (res.v, v), (res.weights, w)):
                assert torch.equal(got[b, h, :n[b]], src[b, h, at])
                assert (got[b, h, n[b]:] == 0).all()


EVICT = [
    # B H C D keep sink recent type layout
    (1, 1, 1, 64, 1, 0, 0, BF, "bhsd"),
    (2, 3, 100, 64, 1, 0, 0, BF, "bhsd"),
    (2, 3, 100, 64, 40, 4, 10, FP, "bshd"),
    (1, 2, 1025, 96, 512, 0, 512, BF, "bhsd"),   # nothing but the recent rows
    (1, 2, 1025, 96, 512, 500, 12, BF, "bhsd"),  # sinks and recent rows only
    (2, 2, 5000, 33, 1111, 4, 64, FP, "bhsd"),   # rows without 16-byte alignment
    (1, 1, 20000, 8, 7000, 4, 64, BF, "bhsd"),
    (3, 1, 64, 128, 64, 0, 0, BF, "bhsd"),       # everything stays
    (2, 2, 50, 16, 80, 4, 4, BF, "bhsd"),        # a budget past the capacity
    (2, 80, 2500, 64, 900, 4, 16, BF, "bhsd"),   # a block per head
    (1, 90, 4096, 40, 1500, 4, 16, FP, "bshd"),  # two blocks per head
    (40, 4, 9000, 8, 700, 2, 30, BF, "bhsd"),    # more keys than a block's registers hold
]


def evict_weights(kind, B, H, C, g):
    w = torch.randn(B, H, C, generator=g).exp()
    if kind == "ties":
        w = torch.randint(0, 3, (B, H, C), generator=g).float()
    elif kind == "equal":
        w = torch.full((B, H, C), 0.25)
    elif kind == "odd":
        pick = torch.randint(0, 6, (B, H, C), generator=g)
        vals = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-42])
        w = vals[pick]
    return w.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=ids)
def test_evict_matches_definition(cuda, case, kind):
    from minference import ops

    B, H, C, D, keep, sink, recent, dtype, layout = case
    g = torch.Generator().manual_seed(9)
    k, v = (cache(g, B, H, C, D, dtype, layout) for _ in range(2))
    w = evict_weights(kind, B, H, C, g)
    res = ops.evict_cache(k, v, w, keep, sink=sink, recent=recent)
    if kind == "odd":  # NaN weights cannot be compared by value
        w2 = w.nan_to_num(nan=-1.0, posinf=9.0, neginf=-9.0)
        res = res._replace(weights=torch.where(res.index < 0, res.weights,
                                               res.weights.nan_to_num(nan=-1.0, posinf=9.0,
                                                                      neginf=-9.0)))
        ref = ref_evict(w, keep, None, sink, recent)
        for b in range(B):
            for h in range(H):
                assert res.index[b, h, :min(keep, C)].tolist() == ref[b][h]
                at = torch.tensor(ref[b][h]).cuda()
                assert torch.equal(res.weights[b, h, :min(keep, C)], w2[b, h, at])
    else:
        check_evicted(res, k, v, w, keep, None, sink, recent)
    lens = [[C, 0, 1][b % 3] if b else C * 3 // 4 for b in range(B)]
    res = ops.evict_cache(k, v, w.nan_to_num(nan=0.5), keep,
                          torch.tensor(lens, dtype=torch.int32).cuda(), sink=sink, recent=recent)
    check_evicted(res, k, v, w.nan_to_num(nan=0.5), keep, lens, sink, recent)


@pytest.mark.gpu
def test_evict_long_cache_selects_past_registers(cuda):
    from minference import ops

    C = 400001
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randn(1, 1, C, 8, generator=g).to(BF).cuda() for _ in range(2))
    w = torch.randint(0, 1000, (1, 1, C), generator=g).float().cuda()
    for keep in (399999, 12345):
        check_evicted(ops.evict_cache(k, v, w, keep, sink=4, recent=64), k, v, w, keep, None, 4, 64)


@pytest.mark.gpu
def test_evict_into_given_buffers(cuda):
    from minference import ops

    g = torch.Generator().manual_seed(11)
    k, v = (cache(g, 2, 2, 300, 64, BF) for _ in range(2))
    w = torch.rand(2, 2, 300, generator=g).cuda()
    buf = torch.full((2, 2, 128, 2, 64), 7.0, dtype=BF, device="cuda")  # [2, B, S, H, D]
    wb = torch.full((2, 2, 130), 7.0, device="cuda")
    ko, vo = buf[0].transpose(1, 2)[:, :, 10:110], buf[1].transpose(1, 2)[:, :, 10:110]
    res = ops.evict_cache(k, v, w, 100, torch.tensor([300, 60]).cuda(), sink=4, recent=8,
                          out=(ko, vo, wb[:, :, 3:103]))
    assert res.k.data_ptr() == ko.data_ptr()
    check_evicted(res, k, v, w, 100, [300, 60], 4, 8)
    assert (buf[:, :, :10] == 7).all() and (buf[:, :, 110:] == 7).all()
    assert (wb[:, :, :3] == 7).all() and (wb[:, :, 103:] == 7).all()


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP])
def test_prefill_evict_and_decode_together(cuda, dtype):
    """A prompt's sparse prefill, the weights of its last queries, its cache cut
    down, then sequences that decode over what is left, weigh their own caches
    and cut those."""
    from minference import ops

    H, S, D, B, keep = 4, 1000, 96, 3, 256
    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn(1, H, S, D, generator=g).to(dtype).cuda() for _ in range(3))
    ops.streaming_forward(q, k, v, 64, 256)
    w = ops.accumulate_attention_weights(q[:, :, -64:], k)
    ref, tol = ref_weights(q[:, :, -64:], k, None)
    assert ((w.double() - ref).abs() <= tol).all()
    pre = ops.evict_cache(k, v, w, keep, sink=4, recent=32)
    check_evicted(pre, k, v, w, keep, None, 4, 32)

    C = 24
    ko, vo = (torch.zeros(B, H, C, D, dtype=dtype, device="cuda") for _ in range(2))
    wo = torch.zeros(B, H, C, device="cuda")
    wref = torch.zeros(B, H, C, dtype=torch.float64, device="cuda")
    wtol = torch.zeros_like(wref)
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    for step in range(20):
        qs, kn, vn = (torch.randn(B, H, 1, D, generator=g).to(dtype).cuda() for _ in range(3))
        ko[:, :, step], vo[:, :, step] = kn[:, :, 0], vn[:, :, 0]
        lens += 1
        out, lse = ops.shared_prefix_attention(qs, pre.k, pre.v, ko, vo, lens, return_lse=True)
        ref, tol, _, _ = ref_attention(qs, pre.k, pre.v, ko, vo, lens.tolist())
        assert ((out.double() - ref).abs() <= tol).all()
        ops.accumulate_attention_weights(qs, ko, wo, lens, lse=lse)
        r, t = ref_weights(qs, ko, None, lens.tolist(), lse=lse)
        wref += r
        wtol += t + 2.0**-23 * wref
    assert ((wo.double() - wref).abs() <= wtol).all()
    cut = ops.evict_cache(ko, vo, wo, 8, lens, sink=1, recent=3)
    check_evicted(cut, ko, vo, wo, 8, lens.tolist(), 1, 3)
    qs = torch.randn(B, H, 1, D, generator=g).to(dtype).cuda()
    out = ops.shared_prefix_attention(qs, pre.k, pre.v, cut.k, cut.v, cut.lengths)
    ref, tol, _, _ = ref_attention(qs, pre.k, pre.v, cut.k, cut.v, cut.lengths.tolist())
    assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_steps_captured_in_graphs_follow_lengths(cuda):
    """Two captured steps replayed with other inputs and lengths, in turn."""
    from minference import ops

    sizes = [(4, 8, 2, 1, 1, 900, 200, 128, BF, "bhsd"), (40, 4, 1, 2, 1, 500, 60, 96, FP, "bhsd")]
    runs = []
    for i, c in enumerate(sizes):
        q, kp, vp, k, v = make(c, 13 + i)
        lens = torch.full((c[0],), c[6], dtype=torch.int32, device="cuda")
        w = torch.zeros(c[0], c[2], c[6], device="cuda")

        def step(q=q, kp=kp, vp=vp, k=k, v=v, lens=lens, w=w):
            o, z = ops.shared_prefix_attention(q, kp, vp, k, v, lens, return_lse=True)
            w.zero_()
            ops.accumulate_attention_weights(q, k, w, lens, lse=z)
            w2 = ops.accumulate_attention_weights(q, k, None, lens)
            e = ops.evict_cache(k, v, w, 32, lens, sink=2, recent=4)
            return o, w2, e

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        runs.append((graph, q, kp, vp, k, v, lens, w, res))
    for turn in range(3):
        for graph, q, kp, vp, k, v, lens, w, (o, w2, e) in runs:
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)))
            lens.copy_(torch.randint(1, k.shape[2] + 1, lens.shape,
                                     generator=torch.Generator().manual_seed(turn + 9)))
        for graph, *_ in runs:
            graph.replay()
        for graph, q, kp, vp, k, v, lens, w, (o, w2, e) in runs:
            ref, tol, _, _ = ref_attention(q, kp, vp, k, v, lens.tolist())
            assert ((o.double() - ref).abs() <= tol).all()
            ref, tol = ref_weights(q, k, None, lens.tolist())
            assert ((w2.double() - ref).abs() <= tol).all()
            check_evicted(e, k, v, w, 32, lens.tolist(), 2, 4)


_FIRST_CALL = """
import sys
sys.path[:0] = [{root!r}, {root!r} + "/minference-npu_b200", {root!r} + "/tests"]
import torch
from minference import ops
import test_cache_ops as t
c = (4, 8, 2, 1, 1, 900, 200, 128, t.BF, "bhsd")
q, kp, vp, k, v = t.make(c, 40)
k2, q2 = k[:, :, :100].contiguous(), q.expand(-1, -1, 70, -1).contiguous()
w = torch.rand(4, 2, 200, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    o = ops.shared_prefix_attention(q, kp, vp, k, v)
    x = ops.accumulate_attention_weights(q2, k2)
    e = ops.evict_cache(k, v, w, 50)
g.replay()
torch.cuda.synchronize()
ref, tol, _, _ = t.ref_attention(q, kp, vp, k, v)
assert ((o.double() - ref).abs() <= tol).all()
ref, tol = t.ref_weights(q2, k2, None)
assert ((x.double() - ref).abs() <= tol).all()
t.check_evicted(e, k, v, w, 50, None, 0, 0)
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_can_be_captured(cuda):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", _FIRST_CALL.format(root=root)], check=True, timeout=240)


@pytest.mark.gpu
def test_streams_and_repeated_calls_agree(cuda):
    """Calls on side streams at once, each equal to the call alone, bit for bit."""
    from minference import ops

    cases = [ATTENTION[2], ATTENTION[7], ATTENTION[9], ATTENTION[11]]
    ins = [make(c, 20) for c in cases]
    alone = [ops.shared_prefix_attention(*x) for x in ins]
    walone = [ops.accumulate_attention_weights(x[0], x[3]) for x in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    for _ in range(3):
        got, wgot = [], []
        for x, s in zip(ins, streams):
            with torch.cuda.stream(s):
                got.append(ops.shared_prefix_attention(*x))
                wgot.append(ops.accumulate_attention_weights(x[0], x[3]))
        torch.cuda.synchronize()
        for a, b in zip(alone + walone, got + wgot):
            assert torch.equal(a, b)
    from minference import _native

    assert _native.device_error() == 0


@pytest.mark.gpu
def test_empty_calls(cuda):
    from minference import ops

    z = torch.zeros(0, 4, 1, 64, dtype=BF, device="cuda")
    kv = torch.zeros(0, 2, 9, 64, dtype=BF, device="cuda")
    assert ops.shared_prefix_attention(z, None, None, kv, kv).shape == z.shape
    assert ops.accumulate_attention_weights(z, kv).shape == (0, 2, 9)
    w = torch.zeros(0, 2, 9, device="cuda")
    assert ops.evict_cache(kv, kv, w, 3).k.shape == (0, 2, 3, 64)
    q = torch.ones(2, 4, 3, 64, dtype=BF, device="cuda")
    e = torch.zeros(2, 2, 0, 64, dtype=BF, device="cuda")
    out, lse = ops.shared_prefix_attention(q, None, None, e, e, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    r = ops.evict_cache(e, e, torch.zeros(2, 2, 0, device="cuda"), 3)
    assert (r.index == -1).all() and (r.lengths == 0).all() and (r.k == 0).all()
    c = torch.ones(2, 2, 5, 64, dtype=BF, device="cuda")
    w = torch.rand(2, 2, 5, device="cuda")
    same = ops.accumulate_attention_weights(q[:, :, :0], c, w.clone())
    assert torch.equal(same, w)
    assert (ops.accumulate_attention_weights(q[:, :, :0], c) == 0).all()


# ---------------------------------------------------------------------------
# Refusals (no GPU: the device check is stepped over, nothing is launched)
# ---------------------------------------------------------------------------


@pytest.fixture
def no_device_check(monkeypatch):
    from minference import _native

    monkeypatch.setattr(_native, "require_cuda", lambda *a: None)

    def never():
        raise AssertionError("a refused call reached the library")

    monkeypatch.setattr(_native, "lib", never)


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    from minference import ops

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.shared_prefix_attention(t(1, 2, 1, 64), None, None, t(1, 2, 8, 64), t(1, 2, 8, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.accumulate_attention_weights(t(1, 2, 1, 64), t(1, 2, 8, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.evict_cache(t(1, 2, 8, 64), t(1, 2, 8, 64), t(1, 2, 8, dtype=torch.float32), 4)


@pytest.mark.parametrize("call, err", [
    (lambda f: f(t(2, 4, 1, 64), None, None, None, None), "neither"),
    (lambda f: f(t(2, 4, 1, 64), t(1, 2, 8, 64), None, None, None), "pairs"),
    (lambda f: f(t(2, 4, 64), None, None, t(2, 2, 8, 64), t(2, 2, 8, 64)), "q must be"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(2, 3, 8, 64), t(2, 3, 8, 64)), "query heads"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(2, 2, 8, 64), t(2, 2, 7, 64)), "v must be"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(3, 2, 8, 64), t(3, 2, 8, 64)), "k must be"),
    (lambda f: f(t(3, 4, 1, 64), t(2, 2, 8, 64), t(2, 2, 8, 64), None, None), "over 2 prefixes"),
    (lambda f: f(t(2, 4, 1, 64), t(1, 2, 8, 64), t(1, 2, 8, 64), None, None,
                 torch.tensor([1, 2])), "lengths without"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(2, 2, 8, 64), t(2, 2, 8, 64),
                 prefix_lengths=torch.tensor([1])), "prefix_lengths without"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(2, 2, 8, 64), t(2, 2, 8, 64),
                 torch.tensor([1, 2, 3])), "lengths must be"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(2, 2, 8, 64), t(2, 2, 8, 64),
                 out=t(2, 4, 2, 64)), "out must be"),
    (lambda f: f(t(2, 4, 1, 64), None, None, t(2, 2, 8, 64), t(2, 2, 8, 64),
                 out=t(1, 4, 1, 64).expand(2, -1, -1, -1)), "overlapping rows"),
])
def test_attention_refuses(no_device_check, call, err):
    from minference import ops

    with pytest.raises(ValueError, match=err):
        call(ops.shared_prefix_attention)


def test_attention_refuses_types_and_overlaps(no_device_check):
    from minference import ops

    f = ops.shared_prefix_attention
    q, c = t(2, 4, 1, 64), t(2, 2, 8, 64)
    with pytest.raises(TypeError):
        f(q.float(), None, None, c.float(), c.float())
    with pytest.raises(TypeError):
        f(q, None, None, c, c.half())
    with pytest.raises(TypeError, match="integer"):
        f(q, None, None, c, c, torch.tensor([1.0, 2.0]))
    with pytest.raises(NotImplementedError, match="head_dim"):
        f(t(2, 4, 1, 136), None, None, t(2, 2, 8, 136), t(2, 2, 8, 136))
    with pytest.raises(ValueError, match="overlaps q"):
        f(q, None, None, c, c, out=q)
    with pytest.raises(ValueError, match="overlaps k"):
        f(q, None, None, c, t(2, 2, 8, 64), out=c.view(2, 4, 4, 64)[:, :, :1])


@pytest.mark.parametrize("cap", [100, 200, 40000, 1 << 20])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64,
                                   torch.uint16, torch.uint32])
def test_lengths_of_every_integer_type(dtype, cap):
    """Types that cannot hold the capacity too: their values are clamped as numbers."""
    from minference.ops._cache import lengths_arg

    values = [0, 1, 99, 127]
    if dtype not in (torch.uint8, torch.uint16, torch.uint32):
        values += [-5, -128]
    if dtype is torch.int64:
        values += [1 << 40, -(1 << 40)]
    got = lengths_arg("lengths", torch.tensor(values, dtype=dtype), len(values), cap,
                      torch.device("cpu"))
    assert got.dtype == torch.int32
    assert got.clamp(0, cap).tolist() == [min(max(x, 0), cap) for x in values]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16])
def test_narrow_lengths_of_a_long_cache(cuda, dtype):
    from minference import ops

    q, _, _, k, v = make((2, 2, 2, 1, 1, 0, 40000, 64, BF, "bhsd"), 37)
    lt, l32 = (torch.tensor([200, 7], dtype=x).cuda() for x in (dtype, torch.int32))
    assert torch.equal(ops.shared_prefix_attention(q, None, None, k, v, lt),
                       ops.shared_prefix_attention(q, None, None, k, v, l32))
    w = ops.accumulate_attention_weights(q, k, None, lt)
    assert torch.equal(w, ops.accumulate_attention_weights(q, k, None, l32))
    assert torch.equal(ops.evict_cache(k, v, w, 50, lt).index,
                       ops.evict_cache(k, v, w, 50, l32).index)


def test_overlap_of_interleaved_views():
    """Views whose elements lie between each other's do not overlap; views that
    share an element always do."""
    import random

    from minference.ops._cache import overlap

    kv = t(2, 4, 10, 128)
    assert not overlap(kv[..., :64], kv[..., 64:])
    assert overlap(kv[..., :65], kv[..., 64:])
    kv = t(3, 2, 4, 10, 64)
    assert not overlap(kv[:, 0], kv[:, 1])
    assert not overlap(kv[:, 0], kv[1, 1])
    assert overlap(kv[:, 0, :, 2:], kv[:, 0, :, :3])
    assert not overlap(kv[:, 1, :, 3:], kv[:, 1, :, :3])
    flat = t(4, 10, 3, 8, 64)  # [B, S, 3, H, D]: a packed projection
    q, k, v = (flat[:, :, i].transpose(1, 2) for i in range(3))
    assert not overlap(q, k) and not overlap(v, q) and overlap(q, q[:, 3:])
    rng = random.Random(1)
    apart = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            size = [rng.randint(1, 4) for _ in range(3)]
            stride = [rng.choice([1, 2, 3, 4, 6, 8, 12, 24]) for _ in range(3)]
            base = torch.arange(400)
            views.append(base.as_strided(size, stride, rng.randint(0, 60)))
        sets = [set(x.flatten().tolist()) for x in views]
        base = torch.arange(400)
        a, b = (base.as_strided(x.shape, x.stride(), x.storage_offset()) for x in views)
        if sets[0] & sets[1]:
            assert overlap(a, b)
        apart += not overlap(a, b)
    assert apart > 1000


@pytest.mark.gpu
def test_interleaved_buffers(cuda):
    """Keys beside values in one buffer, and an output among a packed projection."""
    from minference import ops

    g = torch.Generator().manual_seed(38)
    for shape in ((2, 3, 300, 2, 64), (2, 2, 3, 300, 64)):  # [B,H,S,2,D], [B,2,H,S,D]
        d = shape.index(2, 1)
        kv = torch.randn(shape, generator=g).to(BF).cuda()
        out = torch.full([100 if n == 300 else n for n in shape], 7.0, dtype=BF, device="cuda")
        w = torch.rand(2, 3, 300, generator=g).cuda()
        k, v = kv.unbind(d)
        res = ops.evict_cache(k, v, w, 100, sink=4, recent=8,
                              out=(*out.unbind(d), torch.empty(2, 3, 100, device="cuda")))
        check_evicted(res, k, v, w, 100, None, 4, 8)
    packed = torch.randn(2, 5, 4, 6, 64, generator=g).to(BF).cuda()  # [B, S, q k v o, H, D]
    q, k, v, o = (x.transpose(1, 2) for x in packed.clone().unbind(2))
    ops.shared_prefix_attention(q, None, None, k, v, out=o)
    ref, tol, _, _ = ref_attention(q, None, None, k, v)
    assert ((o.double() - ref).abs() <= tol).all()
    for x, y in zip((q, k, v), packed.unbind(2)):
        assert torch.equal(x, y.transpose(1, 2))


def test_weights_refuse(no_device_check):
    from minference import ops

    f = ops.accumulate_attention_weights
    q, k = t(2, 4, 1, 64), t(2, 2, 8, 64)
    w = t(2, 2, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="weights must be"):
        f(q, k, w[:, :, :7])
    with pytest.raises(TypeError, match="float32"):
        f(q, k, w.half())
    with pytest.raises(ValueError, match="unit stride"):
        f(q, k, t(2, 2, 16, dtype=torch.float32)[:, :, ::2])
    with pytest.raises(ValueError, match="overlapping rows"):
        f(q, k, t(1, 2, 8, dtype=torch.float32).expand(2, -1, -1))
    with pytest.raises(ValueError, match="same view"):
        b = t(2, 2, 9, dtype=torch.float32)
        f(q, k, b[:, :, :8], out=b[:, :, 1:])
    with pytest.raises(ValueError, match="lse must be"):
        f(q, k, w, lse=t(2, 4, dtype=torch.float32))
    with pytest.raises(TypeError, match="lse"):
        f(q, k, w, lse=t(2, 4, 1))
    with pytest.raises(ValueError, match="k must be"):
        f(q, t(2, 2, 8, 32), w)


def test_evict_refuses(no_device_check):
    from minference import ops

    k, v, w = t(2, 2, 8, 64), t(2, 2, 8, 64), t(2, 2, 8, dtype=torch.float32)
    for kw in (dict(keep=0), dict(keep=4, sink=-1), dict(keep=4, sink=3, recent=2)):
        with pytest.raises(ValueError, match="keep"):
            ops.evict_cache(k, v, w, **kw)
    with pytest.raises(ValueError, match="v must be"):
        ops.evict_cache(k, v[:, :1], w, 4)
    with pytest.raises(ValueError, match="weights must be"):
        ops.evict_cache(k, v, w[:, :, :4], 4)
    with pytest.raises(ValueError, match="overlaps"):
        ops.evict_cache(k, v, w, 4, out=(k[:, :, :4], t(2, 2, 4, 64), t(2, 2, 4,
                                                                       dtype=torch.float32)))
    with pytest.raises(ValueError, match="overlaps"):
        o = t(2, 2, 4, 64)
        ops.evict_cache(k, v, w, 4, out=(o, o, t(2, 2, 4, dtype=torch.float32)))
    with pytest.raises(TypeError):
        ops.evict_cache(k.float(), v.float(), w, 4)


def test_c_entry_points_refuse():
    """Status codes of the C entry points, before anything touches a device."""
    from minference import _native, build

    build.build()
    L = _native.lib()
    ok = (1 << 20, 4096, 1024, 64)
    odd = ((1 << 20) + 2, 4096, 1024, 64)    # not 16-byte aligned
    step = (1 << 20, 4096, 1024, 60)         # rows not 16 bytes apart
    flat = (1 << 20, 0, 1024, 64)            # one entry for all
    null = (0, 4096, 1024, 64)
    none = 2**64 - 1

    def attn(q=ok, kp=ok, vp=ok, k=ok, v=ok, out=ok, B=2, Hq=4, Hkv=2, Sq=1, G=2, P=8, C=8, D=64,
             dtype=1, ws=None, n=0, size=False):
        args = _native.SHARED_PREFIX_ARGS.pack(*q, *kp, *vp, *k, *v, *out, 0, 0, 0, B, Hq, Hkv,
                                               Sq, G, P, C, D, dtype, 1, 1.0)
        if size:
            return L.mi_shared_prefix_fwd_workspace_size(args)
        return L.mi_shared_prefix_fwd(args, ws, n, None)

    assert L.mi_shared_prefix_fwd(None, None, 0, None) == 1
    assert attn(dtype=2) == 2
    for bad in (dict(Hq=3), dict(Hkv=0), dict(G=0), dict(B=3, G=2), dict(D=132), dict(D=60), dict(D=24),
                dict(D=0), dict(P=-1), dict(C=-1), dict(C=1 << 31), dict(Sq=-1),
                dict(P=1 << 30, C=64), dict(B=1 << 20, Hq=1 << 20)):
        assert attn(**bad) == 1, bad
        assert attn(size=True, **bad) == none, bad
    assert attn(B=0) == 0 and attn(Sq=0) == 0
    for x in (odd, flat, null):
        for name in ("q", "kp", "vp", "k", "v", "out"):
            assert attn(**{name: x}) == 5, name
    assert attn(k=step) == 5 and attn(vp=step) == 5
    assert attn() == 3 and attn(ws=1 << 20, n=64) == 3  # two segments need a workspace
    assert attn(ws=(1 << 20) + 4, n=1 << 30) == 3
    assert 0 < attn(G=1, P=1000, size=True) < attn(G=1, P=100000, size=True)

    def weights(q=ok, k=ok, lse=0, wo=1 << 20, B=2, Hq=4, Hkv=2, Sq=1, C=8, D=64, dtype=1,
                ws=None, n=0, size=False):
        args = _native.ATTN_WEIGHTS_ARGS.pack(*q, *k, lse, 0, 0, 0, 0, wo, 16, 8, B, Hq, Hkv, Sq,
                                              C, D, dtype, 1, 1.0)
        if size:
            return L.mi_attn_weights_workspace_size(args)
        return L.mi_attn_weights(args, ws, n, None)

    assert L.mi_attn_weights(None, None, 0, None) == 1
    assert weights(dtype=7) == 2
    for bad in (dict(Hq=3), dict(D=136), dict(C=-1), dict(Hkv=0), dict(wo=0), dict(Sq=0)):
        assert weights(**bad) == 1, bad
    assert weights(q=odd) == 5 and weights(k=step) == 5 and weights(k=null) == 5
    assert weights() == 3
    assert weights(B=0) == 0 and weights(C=0) == 0
    assert weights(lse=1 << 20, size=True) == 0 and weights(size=True) > 0

    def evict(k=ok, v=ok, w=1 << 20, ko=ok, vo=ok, wo=1 << 20, idx=1 << 20, nl=1 << 20, B=2, H=2,
              C=8, D=64, keep=4, sink=0, recent=0):
        args = _native.EVICT_ARGS.pack(*k, *v, w, 16, 8, *ko, *vo, wo, 8, 4, idx, nl, 0, B, H, C,
                                       D, keep, sink, recent)
        return L.mi_evict_cache(args, None)

    assert L.mi_evict_cache(None, None) == 1
    for bad in (dict(keep=0), dict(sink=3, recent=2), dict(sink=-1), dict(recent=-1), dict(D=0),
                dict(D=2000), dict(C=-1), dict(idx=0), dict(nl=0), dict(wo=0), dict(w=0),
                dict(k=null), dict(vo=null), dict(sink=2**62, recent=2**62),
                dict(B=1 << 20, H=1 << 20)):
        assert evict(**bad) == 1, bad
    assert evict(B=0) == 0 and evict(H=0) == 0


def test_argument_structs_match_the_header():
    """The packed layouts have the sizes that a C compiler gives the structs."""
    import subprocess
    import tempfile

    from minference import _native

    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = (f'#include "{root}/include/minference_b200.h"\n#include <stdio.h>\n'
           'int main(void){printf("%zu %zu %zu %zu %zu %zu", sizeof(mi_shared_prefix_args), '
           'sizeof(mi_attn_weights_args), sizeof(mi_evict_args), '
           'offsetof(mi_shared_prefix_args, dtype), offsetof(mi_attn_weights_args, dtype), '
           'offsetof(mi_evict_args, B));return 0;}')
    with tempfile.TemporaryDirectory() as d:
        with open(d + "/a.c", "w") as f:
            f.write(src)
        subprocess.check_call(["gcc", "-o", d + "/a", d + "/a.c"])
        got = [int(x) for x in subprocess.check_output([d + "/a"]).split()]
    assert got[:3] == [_native.SHARED_PREFIX_ARGS.size, _native.ATTN_WEIGHTS_ARGS.size,
                       _native.EVICT_ARGS.size]
    assert got[3:] == [8 * 35, 8 * 22, 8 * 25]
