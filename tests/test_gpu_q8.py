"""The 8-bit paged cache on the GPU: the rotating append, decode attention and
the block operations against their plain 64-bit forms (tests/q8_ref.py)."""
import math

import numpy as np
import pytest
import torch

from rvllm_amd.kv_storage import HipGatherPlan, HipKvStorage
from rvllm_amd.q8_storage import HipQ8Storage
from tests import q8_ref as ref
from tests.q8_ref import i32

pytestmark = pytest.mark.gpu

F = {"f16": torch.float16, "f32": torch.float32}


def randn(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * scale


def slots(rows, nb, bs, seed):
    """rows distinct slots anywhere in the pool."""
    at = np.random.default_rng(seed).permutation(nb * bs)[:rows]
    return at // bs, at % bs


def inv_freq(rot, base=1e6):
    return torch.from_numpy((base ** (-np.arange(0, rot, 2) / rot)
                             ).astype(np.float32)).cuda()


# -- append -------------------------------------------------------------------

APPENDS = [
    # H, kv, hd, bs, rot, interleaved, dtype, rows, fused
    (32, 8, 64, 16, 64, False, "f16", 1, True),
    (15, 5, 64, 16, 32, True, "f32", 37, True),
    (16, 8, 128, 16, 128, False, "f16", 131, True),
    (16, 8, 128, 32, 64, False, "f32", 50, False),
    (4, 1, 256, 16, 256, False, "f16", 33, True),
    (4, 1, 256, 48, 64, True, "f16", 5, False),
    (4, 2, 32, 16, 32, False, "f32", 9, True),
    (6, 2, 80, 48, 80, False, "f16", 40, True),     # 16 lanes a head
    (6, 2, 80, 16, 20, True, "f32", 40, True),
    (3, 3, 112, 16, 112, False, "f16", 21, True),
    (9, 3, 192, 16, 96, False, "f32", 17, True),
    (2, 1, 16, 16, 16, False, "f32", 3, True),
    (8, 2, 64, 16, 24, False, "f16", 19, True),     # rot / 2 not in eights
    (8, 2, 64, 16, 0, False, "f16", 19, True),      # no rotation
    (4, 2, 128, 16, 128, False, "f16", 2050, True),  # four tokens a workgroup
    (3, 1, 80, 32, 48, True, "f32", 2051, True),
]


def append_inputs(H, kv, hd, rows, dtype, fused, seed):
    x = (randn((rows, (H + 2 * kv) * hd), seed)
         * torch.exp2(randn(((H + 2 * kv) * hd,), seed + 1))).to(F[dtype])
    q, k, v = (t.view(rows, -1, hd) for t in
               x.split([H * hd, kv * hd, kv * hd], dim=1))
    return (q, k, v) if fused else tuple(t.contiguous() for t in (q, k, v))


@pytest.mark.parametrize("H,kv,hd,bs,rot,inter,dtype,rows,fused", APPENDS)
@pytest.mark.parametrize("norm", [False, True])
def test_q8_rope_append(H, kv, hd, bs, rot, inter, dtype, rows, fused, norm):
    nb = -(-rows // bs) + 3
    st = HipQ8Storage(2, nb, bs, kv, hd)
    q, k, v = append_inputs(H, kv, hd, rows, dtype, fused, 11)
    pos = np.random.default_rng(5).integers(0, 1 << 21, rows)
    pos[0] = (1 << 32) - 1  # the farthest there is
    blk, off = slots(rows, nb, bs, 7)
    wq, wk = ((1 + randn(hd, 3) * 0.2, 1 + randn(hd, 4) * 0.2) if norm
              else (None, None))
    inv = inv_freq(rot) if rot else None
    got = st.rope_append(1, q, k, v, i32(pos), inv, i32(blk), i32(off),
                         interleaved=inter, attn_factor=1.13, q_norm=wq,
                         k_norm=wk, eps=1e-6)
    f32f = float(np.float32(1.13))
    eps = float(np.float32(1e-6))
    want_q = ref.rotate(q, pos, inv, inter, f32f, wq, eps)
    want_k = ref.rotate(k, pos, inv, inter, f32f, wk, eps)
    # q is rounded once: half a step of its type, and for the sums and angles
    # before it 2^-40 of its row's largest value in f64, 2^-21 (eight roundings
    # of 2^-24: angles, norm, weight, products, sum) where f16 q takes f32
    before = 2.0 ** (-21 if q.dtype == torch.float16 else -40)
    room = (torch.finfo(q.dtype).eps / 2 * 1.0001 * want_q.abs()
            + 2.0 ** -24 * torch.finfo(q.dtype).tiny
            + before * want_q.abs().amax(-1, keepdim=True)
            + (2.0 ** -25 if q.dtype == torch.float16 else 0))
    assert ((got.cpu().double() - want_q).abs() <= room).all()
    for which, x in ((0, want_k), (1, v.double().cpu())):
        codes, scale = ref.quantise(x)
        gc = st.codes(1, which).cpu()[blk, :, off]
        gs = st.scales(1, which).cpu()[blk, :, off]
        assert torch.equal(gc, codes)
        assert torch.equal(gs, scale)
    # every other slot and the other layer stay as they were
    assert not st.codes(0, 0).any() and not st.codes(0, 1).any()
    for which in (0, 1):
        rest = st.scales(1, which).clone()
        rest[torch.from_numpy(blk).cuda(), :, torch.from_numpy(off).cuda()] = 0
        assert not rest.any()


@pytest.mark.parametrize("cell", ["f16", "f32"])
@pytest.mark.parametrize("H,kv,hd,bs,rot,inter,dtype,rows,fused", APPENDS)
def test_rope_append_into_f16_and_f32_pools(H, kv, hd, bs, rot, inter, dtype,
                                            rows, fused, cell):
    nb = -(-rows // bs) + 2
    st = HipKvStorage(2, nb, bs, kv, hd, dtype=F[cell])
    q, k, v = append_inputs(H, kv, hd, rows, dtype, fused, 21)
    pos = np.random.default_rng(6).integers(0, 1 << 20, rows)
    blk, off = slots(rows, nb, bs, 8)
    inv = inv_freq(rot) if rot else None
    got = st.rope_append(1, q, k, v, i32(pos), inv, i32(blk), i32(off),
                         interleaved=inter)
    want_q = ref.rotate(q, pos, inv, inter, 1.0)
    assert ((got.cpu().double() - want_q).abs()
            <= torch.finfo(q.dtype).eps / 2 * 1.0001 * want_q.abs()
            + 2.0 ** -21 * want_q.abs().amax(-1, keepdim=True)
            + 2.0 ** -24).all()
    for which, x in ((0, ref.rotate(k, pos, inv, inter, 1.0)),
                     (1, v.double().cpu())):
        cells = st.read_blocks(1, which, i32(np.arange(nb))).cpu()
        have = cells[blk, off].double()  # [rows, kv, hd]
        assert ((have - x).abs() <= torch.finfo(F[cell]).eps / 2 * 1.0001
                * x.abs() + 2.0 ** -25).all()


def test_q8_append_rows_that_are_special():
    """Zeros, one value, ties of a code's border, rows that are not finite,
    the largest and the smallest magnitudes."""
    hd, bs = 64, 16
    st = HipQ8Storage(1, 2, bs, 1, hd)
    x = torch.zeros((8, 1, hd))
    x[1, 0, 5] = -3.0
    x[2, 0] = torch.arange(hd) * 0.5  # scale 31.5 / 127, borders between
    x[3, 0, :] = 1.0
    x[3, 0, 9] = math.nan
    x[4, 0, 3] = math.inf
    x[5, 0] = 3.0e38
    x[6, 0] = 1e-42
    x[6, 0, 1] = -2e-44
    x[7, 0] = torch.arange(hd) + 0.5  # scale 0.5: every value a tie or whole
    x[7, 0, 63] = 63.5
    v = x.flip(0).contiguous()
    n = np.arange(8)
    st.write_tokens(0, i32(n * 0), i32(n), x.cuda(), v.cuda())
    for which, y in ((0, x), (1, v)):
        codes, scale = ref.quantise(y.double())
        assert torch.equal(st.codes(0, which)[0, 0, :8].cpu(), codes[:, 0])
        got = st.scales(0, which)[0, 0, :8].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(scale[:, 0]))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(scale[:, 0]))


def test_q8_append_skips_slots_out_of_range():
    st = HipQ8Storage(1, 3, 16, 2, 64)
    q = randn((4, 4, 64), 1).half()
    k = randn((4, 2, 64), 2).half()
    blk, off = [3, 0xFFFFFFFF, 1, 2], [0, 0, 16, 5]
    inv = inv_freq(64)
    got = st.rope_append(0, q, k, k, i32([0, 1, 2, 3]), inv, i32(blk),
                         i32(off))
    want = ref.rotate(q, [0, 1, 2, 3], inv, False, 1.0)
    assert (got.cpu().double() - want).abs().max() < 2.0 ** -9
    left = st.scales(0, 0).clone()
    assert left[2, :, 5].all()
    left[2, :, 5] = 0
    assert not left.any()


@pytest.mark.parametrize("first", [0, 1, 3, 14])
def test_q8_append_runs_of_slots(first):
    """Prompts in consecutive slots from any offset on, block ends inside a
    group of four tokens, a slot out of range and one out of order."""
    kv, hd, bs, rows = 2, 64, 16, 2052
    nb = rows // bs + 2
    st = HipQ8Storage(1, nb, bs, kv, hd)
    k, v = randn((rows, kv, hd), 1), randn((rows, kv, hd), 2)
    at = first + np.arange(rows)
    at[[100, 101]] = at[[101, 100]]
    blk, off = at // bs, at % bs
    blk[333] = nb
    st.write_tokens(0, i32(blk), i32(off), k, v)
    keep = np.arange(rows) != 333
    for which, x in ((0, k), (1, v)):
        codes, scale = ref.quantise(x.double().cpu()[keep])
        assert torch.equal(st.codes(0, which).cpu()[blk[keep], :, off[keep]],
                           codes)
        assert torch.equal(st.scales(0, which).cpu()[blk[keep], :, off[keep]],
                           scale)
        assert (st.scales(0, which) != 0).sum() == (rows - 1) * kv


def test_q8_pool_refuses_host_memory():
    from rvllm_amd._lib import RvkvError
    for pin in (False, True):
        mem = torch.zeros(1 << 16, dtype=torch.uint8, pin_memory=pin)
        at = -mem.data_ptr() % 256
        with pytest.raises(RvkvError, match="not the current device's"):
            HipQ8Storage(1, 2, 16, 1, 64, memory=mem[at:])


# -- decode -------------------------------------------------------------------

def filled(nb, bs, kv, hd, seed, layers=1):
    """A pool whose every slot holds quantised N(0, 1) rows of magnitudes that
    differ from row to row."""
    st = HipQ8Storage(layers, nb, bs, kv, hd)
    n = np.arange(nb * bs)
    k, v = (randn((nb * bs, kv, hd), seed + i)
            * torch.exp2(randn((nb * bs, kv, 1), seed + 9 + i))
            for i in (0, 1))
    st.write_tokens(layers - 1, i32(n // bs), i32(n % bs), k, v)
    return st


def dense(st, layer, blocks, n):
    """K and V of a sequence's first n keys, f64 [n, kv, hd], and whether each
    key's block is readable."""
    ok = torch.tensor([b < st.num_blocks for b in blocks])
    at = torch.tensor([int(b) if b < st.num_blocks else 0 for b in blocks])
    got = []
    for which in (0, 1):
        x = (st.codes(layer, which).cpu()[at].double()
             * st.scales(layer, which).cpu()[at].double()[..., None])
        got.append(x.transpose(1, 2).reshape(-1, st.n_kv_heads,
                                             st.head_dim)[:n])
    return got[0], got[1], ok.repeat_interleave(st.block_size)[:n]


def decode_case(H, kv, hd, bs, dtype, ctx, window=0, bad=(), max_ctx=None,
                seed=0, amp=1.0):
    need = [max(1, -(-c // bs)) for c in ctx]
    nb = sum(need) + 2
    st = filled(nb, bs, kv, hd, 100 + seed)
    ids = np.random.default_rng(seed).permutation(nb)
    at = np.cumsum([0] + need)
    tables = [ids[a:a + n].astype(np.int64) for a, n in zip(at, need)]
    for s, j, value in bad:
        tables[s][j] = value
    wide = max(need)
    padded = np.array([list(t) + [t[-1]] * (wide - len(t)) for t in tables])
    q = (randn((len(ctx), H, hd), 300 + seed) * amp).to(F[dtype])
    out = torch.full_like(q, math.nan)
    top = max_ctx or max(max(ctx), 1)
    got = st.paged_decode(0, q, i32(padded), i32(ctx), top, out=out,
                          window=window)
    again = st.paged_decode(0, q, i32(padded), i32(ctx), top, window=window)
    assert torch.equal(got, again)  # no atomics
    for b, c in enumerate(ctx):
        c = min(c, top)
        k, v, ok = dense(st, 0, tables[b], c)
        j = torch.arange(c)
        seen = ok & (j > c - 1 - window if window else j >= 0)
        want, tol = ref.attend(q[b:b + 1], k, v, seen[None], hd ** -0.5)
        ref.check_close(got[b:b + 1], want, tol, f"sequence {b} of {c}")
    return st


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("H,kv,hd,bs", [
    (15, 5, 64, 16), (32, 8, 64, 16), (16, 8, 128, 16), (14, 2, 64, 32),
    (4, 1, 256, 16), (12, 4, 80, 48), (9, 3, 192, 16), (22, 2, 128, 64),
    (2, 2, 16, 16), (40, 2, 48, 32), (8, 1, 240, 16)])
def test_q8_decode_shapes(H, kv, hd, bs, dtype):
    """Lengths around tiles, partitions and nothing at all."""
    decode_case(H, kv, hd, bs, dtype, [1, 0, 15, 16, 17, 63, 64, 65, 300])


@pytest.mark.parametrize("ctx", [[255, 256, 257], [1023, 1024, 1025, 1],
                                 [3000, 2, 777], [5000]])
@pytest.mark.parametrize("window", [0, 1, 33, 600])
def test_q8_decode_partitions_and_windows(ctx, window):
    decode_case(8, 2, 64, 16, "f32", ctx, window=window)
    decode_case(4, 2, 128, 32, "f16", ctx, window=window, seed=1)


def test_q8_decode_bad_blocks_are_left_out():
    decode_case(8, 2, 64, 16, "f32", [100, 40, 16, 700],
                bad=[(0, 1, 1 << 20), (0, 6, 0xFFFFFFFF), (1, 0, 99999),
                     (2, 0, 77777), (3, 20, 55555)])


def test_q8_decode_bound_below_the_lengths():
    decode_case(8, 2, 64, 16, "f32", [500, 20, 300], max_ctx=256)


@pytest.mark.parametrize("amp", [1e-3, 30.0, 3000.0])
def test_q8_decode_magnitudes(amp):
    """Queries far from 1: nearly equal weights, and a single one."""
    decode_case(16, 8, 128, 16, "f32", [400, 64, 2], amp=amp)


def test_q8_decode_masked_cells_are_not_read_as_values():
    """NaN rows behind the context, before the window and in no table leave
    the result; one inside it makes its head NaN."""
    bs, kv, hd = 16, 2, 64
    st = filled(8, bs, kv, hd, 5)
    q = randn((1, 4, hd), 6)
    table, ctx = i32([[0, 1, 2, 3]]), i32([40])
    want = st.paged_decode(0, q, table, ctx, 64, window=20)
    bad = torch.full((1, kv, hd), math.nan, device="cuda")
    for pos in [0, 10, 19, 40, 47, 63, 100]:
        st.write_tokens(0, i32([pos // bs]), i32([pos % bs]), bad, bad)
    assert torch.equal(st.paged_decode(0, q, table, ctx, 64, window=20), want)
    st.write_tokens(0, i32([1]), i32([9]), bad, bad)
    assert torch.isnan(st.paged_decode(0, q, table, ctx, 64, window=20)).all()


def test_q8_decode_values_of_very_different_size():
    """V rows of 2^-100 beside 2^100, in either order of the tiles, zero rows
    among them."""
    bs, hd = 16, 64
    for flip in (False, True):
        st = HipQ8Storage(1, 40, bs, 1, hd)
        n = np.arange(640)
        k = randn((640, 1, hd), 1, 0.1)
        v = randn((640, 1, hd), 2)
        e = torch.linspace(-100, 100, 640, device="cuda").round()
        v = v * torch.exp2(e.flip(0) if flip else e)[:, None, None]
        v[100:180] = 0
        st.write_tokens(0, i32(n // bs), i32(n % bs), k, v)
        q = randn((1, 1, hd), 3)
        got = st.paged_decode(0, q, i32([np.arange(40)]), i32([640]), 640)
        kd, vd, _ = dense(st, 0, list(range(40)), 640)
        want, tol = ref.attend(q, kd, vd, torch.ones(1, 640, dtype=torch.bool),
                               hd ** -0.5)
        ref.check_close(got, want, tol)


# -- gather, copy -------------------------------------------------------------

@pytest.mark.parametrize("kv,hd,bs", [(2, 64, 16), (1, 80, 48), (3, 128, 32)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_q8_gather_and_copy(kv, hd, bs, dtype):
    st = filled(9, bs, kv, hd, 3, layers=2)
    st.copy_blocks(i32([2, 5, 100]), i32([7, 0, 1]))
    for which in (0, 1):
        for a, b in ((2, 7), (5, 0)):
            assert torch.equal(st.codes(1, which)[a], st.codes(1, which)[b])
            assert torch.equal(st.scales(1, which)[a], st.scales(1, which)[b])
    n = 2 * bs + 5
    plan = HipGatherPlan([([7, 3, 4], n), ([1, 500, 2], bs)])
    ok, ov = (torch.empty((2, kv, n, hd), dtype=F[dtype], device="cuda")
              for _ in range(2))
    st.gather(1, plan, ok, ov)
    for b, t in enumerate(([7, 3, 4], [1, 500, 2])):
        k, v, good = dense(st, 1, t, n)
        for got, x in ((ok, k), (ov, v)):
            # code * scale (exact in f64), rounded: half a step of the type,
            # by way of an f32 or not
            x = torch.where(good[:, None, None], x, 0.0)
            err = (got[b].cpu().transpose(0, 1).double() - x).abs()
            assert (err <= (torch.finfo(F[dtype]).eps / 2 + 2.0 ** -24)
                    * x.abs() + 2.0 ** -25).all()


# -- packed prompts -----------------------------------------------------------

def prefill_case(H, kv, hd, bs, dtype, seqs, window=0, bad=(), seed=0,
                 amp=1.0, pad=0, wide_by=0):
    """seqs: (rows, pos_offset, read_num_tokens). pad: rows behind the last
    sequence, which stay as they were."""
    need = [max(1, -(-r // bs)) for _, _, r in seqs]
    nb = sum(need) + 2
    st = filled(nb, bs, kv, hd, 400 + seed)
    ids = np.random.default_rng(seed).permutation(nb)
    at = np.cumsum([0] + need)
    tables = [ids[a:a + n].astype(np.int64) for a, n in zip(at, need)]
    for s, j, value in bad:
        tables[s][j] = value
    wide = max(need) + wide_by
    padded = np.array([list(t) + [t[-1]] * (wide - len(t)) for t in tables])
    starts = np.cumsum([0] + [n for n, _, _ in seqs])
    rows = int(starts[-1]) + pad
    q = (randn((rows, H, hd), 500 + seed) * amp).to(F[dtype])
    out = torch.full_like(q, 7.0)
    args = (0, q, i32(starts), i32(padded), i32([o for _, o, _ in seqs]),
            i32([r for _, _, r in seqs]))
    st.packed_prefill(*args, out=out, window=window)
    again = st.packed_prefill(*args, window=window)
    assert torch.equal(out[:rows - pad], again[:rows - pad])
    assert (out[rows - pad:] == 7.0).all()
    for b, (n, off, read) in enumerate(seqs):
        r = slice(int(starts[b]), int(starts[b + 1]))
        k, v, ok = dense(st, 0, tables[b], read)
        j, pos = torch.arange(read)[None], off + torch.arange(n)[:, None]
        seen = ok[None] & (j <= pos)
        if window:
            seen = seen & (j + window > pos)
        want, tol = ref.attend(q[r], k, v, seen, hd ** -0.5)
        if dtype == "f16":
            # the weights are rounded once to f16 (half a step, or the smallest
            # one of a value of at least half the largest: 2^-25)
            top = torch.where(seen, 1.0, 0.0)
            vmax = v.abs().amax() if read else torch.tensor(0.0)
            tol = tol + vmax * (2.0 ** -11 + 2.0 ** -24
                                * top.sum(-1, keepdim=True).double())
        ref.check_close(out[r], want, tol, f"sequence {b}: {n} rows")
    return st


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("H,kv,hd,bs", [
    (15, 5, 64, 16), (32, 8, 64, 16), (16, 8, 128, 16), (14, 2, 64, 32),
    (4, 1, 256, 16), (12, 4, 80, 48), (9, 3, 192, 16), (22, 2, 128, 64),
    (2, 2, 16, 16), (40, 2, 48, 32), (8, 1, 240, 16)])
def test_q8_packed_prefill_shapes(H, kv, hd, bs, dtype):
    prefill_case(H, kv, hd, bs, dtype,
                 [(1, 0, 1), (63, 0, 63), (0, 0, 0), (130, 0, 130),
                  (5, 200, 205), (64, 7, 71)], pad=3)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("window", [1, 20, 64, 200])
def test_q8_packed_prefill_windows(window, dtype):
    prefill_case(4, 2, 64, 16, dtype, [(300, 0, 300), (90, 333, 423),
                                       (1, 500, 501)], window=window)
    prefill_case(4, 1, 256, 16, dtype, [(100, 0, 100), (40, 50, 90)],
                 window=window, seed=1)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_q8_packed_prefill_reads_and_bad_blocks(dtype):
    """Rows before and behind the read keys, blocks that cannot be read, rows
    that see nothing, a table wider than the context."""
    prefill_case(8, 2, 64, 16, dtype,
                 [(50, 0, 20), (30, 100, 60), (70, 0, 70), (10, 0, 0),
                  (40, 300, 340)],
                 bad=[(0, 0, 1 << 30), (2, 2, 5000), (4, 3, 0xFFFFFFFF)],
                 wide_by=9)
    prefill_case(8, 2, 64, 16, dtype, [(20, 500, 100)], window=50)


@pytest.mark.parametrize("amp", [1e-3, 30.0, 3000.0])
def test_q8_packed_prefill_magnitudes(amp):
    prefill_case(4, 2, 128, 16, "f32", [(140, 0, 140), (20, 300, 320)],
                 amp=amp)


def test_q8_packed_prefill_many_sequences():
    rng = np.random.default_rng(3)
    prefill_case(4, 2, 64, 16, "f16",
                 [(int(n), int(o), int(n + o)) for n, o in
                  zip(rng.integers(0, 20, 300), rng.integers(0, 40, 300))])


def test_q8_packed_prefill_masked_cells_are_not_read_as_values():
    bs, kv, hd = 16, 2, 64
    st = filled(8, bs, kv, hd, 5)
    q = randn((60, 4, hd), 6)
    args = (i32([0, 60]), i32([[0, 1, 2, 3, 4]]), i32([0]), i32([60]))
    want = st.packed_prefill(0, q, *args, window=20)
    bad = torch.full((1, kv, hd), math.nan, device="cuda")
    for pos in [60, 61, 79]:
        st.write_tokens(0, i32([pos // bs]), i32([pos % bs]), bad, bad)
    assert torch.equal(st.packed_prefill(0, q, *args, window=20), want)
    # a NaN row at 30: rows 30 .. 49 see it, and no other
    st.write_tokens(0, i32([1]), i32([14]), bad, bad)
    got = st.packed_prefill(0, q, *args, window=20)
    assert torch.isnan(got[30:50]).all()
    assert torch.equal(got[:30], want[:30])
    assert torch.equal(got[50:], want[50:])


def test_q8_packed_prefill_takes_bad_row_starts():
    """Entries past the rows and decreasing ones: nothing outside is read or
    written."""
    st = filled(8, 16, 2, 64, 5)
    q = randn((40, 4, 64), 6)
    out = torch.full_like(q, 7.0)
    st.packed_prefill(0, q, i32([0, 1 << 31, 30, 0xFFFFFFFF]),
                      i32([[0, 1, 2]] * 3), i32([0] * 3), i32([40] * 3),
                      out=out)
    assert torch.isfinite(out).all()


def test_q8_append_then_prompt_then_decode():
    """The operators as a serving step uses them, against the same steps in 64
    bits: two prompts packed, then three decode steps."""
    H, kv, hd, bs, rot = 8, 2, 64, 16, 32
    st = HipQ8Storage(1, 20, bs, kv, hd)
    inv = inv_freq(rot, 1e4)
    lens, tables = [37, 90], [[3, 7, 1, 15], [2, 5, 8, 11, 14, 17, 19]]
    wide = 7
    padded = i32([t + [t[-1]] * (wide - len(t)) for t in tables])
    held = [[], []]
    n = sum(lens)

    def append(b_of, pos, seed):
        x = randn((len(pos), (H + 2 * kv) * hd), seed).half()
        q, k, v = (t.view(len(pos), -1, hd) for t in
                   x.split([H * hd, kv * hd, kv * hd], dim=1))
        blk = [tables[b][p // bs] for b, p in zip(b_of, pos)]
        off = [p % bs for p in pos]
        got = st.rope_append(0, q, k, v, i32(pos), inv, i32(blk), i32(off),
                             interleaved=True)
        kk = ref.rotate(k, pos, inv, True, 1.0)
        for i, b in enumerate(b_of):
            c, s = zip(ref.quantise(kk[i]), ref.quantise(v[i].double().cpu()))
            held[b].append([ci.double() * si.double()[:, None]
                            for ci, si in zip(c, s)])
        return got

    def want(b, q, first):
        k, v = (torch.stack([h[i] for h in held[b]]) for i in (0, 1))
        pos = first + torch.arange(q.shape[0])[:, None]
        return ref.attend(q, k, v, torch.arange(len(held[b]))[None] <= pos,
                          hd ** -0.5)

    q = append([0] * 37 + [1] * 90, list(range(37)) + list(range(90)), 1)
    out = st.packed_prefill(0, q, i32([0, 37, n]), padded, i32([0, 0]),
                            i32(lens))
    for b, r in ((0, slice(0, 37)), (1, slice(37, n))):
        w, tol = want(b, q[r], 0)
        ref.check_close(out[r], w, tol + 2.0 ** -11 * 6, "prompt")
    for step in range(3):
        pos = [37 + step, 90 + step]
        q = append([0, 1], pos, 10 + step)
        out = st.paged_decode(0, q, padded, i32([p + 1 for p in pos]), 112)
        for b in (0, 1):
            w, tol = want(b, q[b:b + 1], pos[b])
            ref.check_close(out[b:b + 1], w, tol, "decode")


# -- streams, graphs ----------------------------------------------------------

def test_q8_graph_replays_like_eager():
    """Append, packed prompts and decode captured into one graph on a stream
    of its own; replayed beside eager work, each replay with new inputs gives
    the eager bits."""
    H, kv, hd, bs, n = 8, 2, 64, 16, 150
    nb = 40
    st, eager = (HipQ8Storage(1, nb, bs, kv, hd) for _ in range(2))
    inv = inv_freq(hd)
    table = i32([list(range(0, 12)), list(range(12, 24))])
    pos = np.concatenate([np.arange(n), np.arange(n)])
    blk = i32(np.concatenate([pos[:n] // bs, pos[n:] // bs + 12]))
    off, pos = i32(pos % bs), i32(pos)
    starts, zero, reads = i32([0, n, 2 * n]), i32([0, 0]), i32([n, n])
    x = randn((2 * n, (H + 2 * kv) * hd), 1).half()
    out = torch.empty((2 * n, H, hd), dtype=torch.float16, device="cuda")
    dec = torch.empty((2, H, hd), dtype=torch.float16, device="cuda")
    qo = torch.empty_like(out)
    wsp = torch.empty(max(256, st.prefill_workspace_bytes(2 * n, 2, H, 12)),
                      dtype=torch.uint8, device="cuda")
    wsd = st.alloc_workspace(2, H, n)

    def run(s, o, d):
        q, k, v = (t.view(2 * n, -1, hd) for t in
                   x.split([H * hd, kv * hd, kv * hd], dim=1))
        s.rope_append(0, q, k, v, pos, inv, blk, off, q_out=qo)
        s.packed_prefill(0, qo, starts, table, zero, reads, out=o, ws=wsp)
        s.paged_decode(0, o[:2], table, reads, n, out=d, ws=wsd)

    run(st, out, dec)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        st.set_stream(torch.cuda.current_stream())
        run(st, out, dec)
    st.set_stream(torch.cuda.current_stream())
    for seed in range(4):
        x.copy_(randn(x.shape, 50 + seed).half())
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        o2, d2 = torch.empty_like(out), torch.empty_like(dec)
        run(eager, o2, d2)
        torch.cuda.synchronize()
        assert torch.equal(out, o2) and torch.equal(dec, d2)
        assert torch.equal(st.codes(0, 1), eager.codes(0, 1))


def test_q8_pool_on_its_own_stream():
    """Calls run on the pool's stream, whatever torch's current one is."""
    side = torch.cuda.Stream()
    st = filled(40, 16, 2, 64, 3)
    q, table, ctx = randn((2, 4, 64), 1), i32([[3, 5, 7], [9, 11, 2]]), i32(
        [40, 33])
    want = st.paged_decode(0, q, table, ctx, 48)
    torch.cuda.synchronize()
    st.set_stream(side)
    got = torch.zeros_like(want)
    torch.cuda.synchronize()
    st.paged_decode(0, q, table, ctx, 48, out=got)
    side.synchronize()
    assert torch.equal(got, want)


def test_q8_two_calls_at_once_with_their_own_workspaces():
    """Two pools' decodes on two streams, many partitions each."""
    a, b = filled(300, 16, 2, 64, 3), filled(300, 16, 2, 64, 4)
    table, ctx = i32([list(range(300))]), i32([4800])
    q = randn((1, 8, 64), 1)
    want = [s.paged_decode(0, q, table, ctx, 4800) for s in (a, b)]
    ws = [s.alloc_workspace(1, 8, 4800) for s in (a, b)]
    outs = [[torch.empty_like(q) for _ in range(8)] for _ in (a, b)]
    torch.cuda.synchronize()
    for s in (a, b):
        s.set_stream(torch.cuda.Stream())
    for i in range(8):
        for s, w, o in zip((a, b), ws, outs):
            s.paged_decode(0, q, table, ctx, 4800, out=o[i], ws=w)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(x, w) for x in o)


# -- the engine's backend -----------------------------------------------------

def engine_items(rng, vocab, lens, bs, width):
    from rvllm_amd.engine import BatchItem
    items = []
    for i, n in enumerate(lens):
        blocks = list(range(i * width, i * width + width))
        items.append(BatchItem(i, rng.integers(0, vocab, n).tolist(),
                               [(blocks[p // bs], p % bs) for p in range(n)],
                               blocks, n, 0))
    return items


@pytest.mark.parametrize("variant", ["plain", "norm", "bias", "window"])
def test_q8_backend_forward(variant):
    """Prompts in one forward give each prompt's own logits, and a decode step
    those of the prompt with its token (a row's cells depend on the row
    alone): the same f32 computation in another order of sums. Two layers of
    f32 products of 128: 1e-4 of the logits' size is far above their
    rounding."""
    from rvllm_amd.attn_model import AttnModelConfig, HipBackend, init_weights
    from rvllm_amd.engine import BatchItem
    cfg = AttnModelConfig(vocab=256, hidden=128, n_layers=2, n_heads=8,
                          n_kv_heads=2, head_dim=64,
                          qkv_bias=variant == "bias",
                          qk_norm=variant == "norm",
                          window=24 if variant == "window" else 0)
    w = init_weights(cfg)
    rng = np.random.default_rng(1)
    items = engine_items(rng, cfg.vocab, [40, 7, 99], 16, 8)
    be = HipBackend(cfg, w, 30, 16, cache="q8")
    ids = be.forward_sample(items, True, [None] * 3)
    packed = be.last_logits.clone()
    size = packed.abs().max().item()
    for i, it in enumerate(items):
        alone = HipBackend(cfg, w, 30, 16, cache="q8")
        assert alone.forward_sample([it], True, [None]) == [ids[i]]
        assert (alone.last_logits[0] - packed[i]).abs().max() < 1e-4 * size
    step = [BatchItem(it.seq_id, [t], [(it.read_blocks[n // 16], n % 16)],
                      it.read_blocks, n + 1, n)
            for it, t in zip(items, ids) for n in [len(it.tokens)]]
    be.forward_sample(step, False, [None] * 3)
    for i, (it, t) in enumerate(zip(items, ids)):
        n = len(it.tokens) + 1
        whole = HipBackend(cfg, w, 30, 16, cache="q8")
        whole.forward_sample(
            [BatchItem(0, it.tokens + [t],
                       [(it.read_blocks[p // 16], p % 16) for p in range(n)],
                       it.read_blocks, n, 0)], True, [None])
        assert (whole.last_logits[0] - be.last_logits[i]).abs().max() \
            < 1e-4 * size


def test_q8_engine_runs_with_preemption_and_prefix_hits():
    """The engine over the 8-bit backend: preempted requests and shared
    prefixes end with the tokens of an engine with room for all."""
    from rvllm_amd.attn_model import AttnModelConfig, HipBackend, init_weights
    from rvllm_amd.engine import EngineConfig, RequestSpec, run
    cfg = AttnModelConfig(vocab=512, hidden=128, n_layers=2, n_heads=8,
                          n_kv_heads=2, head_dim=64, context_length=512)
    w = init_weights(cfg)
    rng = np.random.default_rng(5)
    shared = rng.integers(0, 512, 40).tolist()
    reqs = [RequestSpec((shared if i % 2 == 0 else []) + rng.integers(
        0, 512, 10 + i).tolist(), 12 + i) for i in range(6)]
    got = [run(HipBackend(cfg, w, n, 16, cache="q8"), reqs,
               EngineConfig(16, n, max_running=6)) for n in (12, 100)]
    assert got[0].generated == got[1].generated
    assert got[0].stats.preemptions > 0 and got[0].stats.prefix_hits > 0
