"""The MXFP8 latent cache, attention over it and draft verification through the C ABI, against oracles in 64 bits."""
import numpy as np
import pytest

import k3o
from latent_util import (LATENT, MX8_PAGE, PAGE, ROPE_AT, ROW, SCALES_AT, attn_oracle, attn_tolerance, bf16_rows, mx8_range_tolerance, mx8_rows, put_rows,
                         quant_rows, verify_oracle)
from util import bf16_bits, normal_bf16, rng, to_dev, to_dev_bf16

pytestmark = pytest.mark.gpu


# ---- cache ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,stride,layers", [(1, 576, 1), (5, 2112, 2), (64, 576, 3), (65, 584, 1), (1027, 576, 2), (300, 5184, 1)])
def test_store(k3g, dev, T, stride, layers):
    import torch
    g = rng(T + stride)
    pages = T // PAGE + 2
    rows = normal_bf16(g, (T, stride), std=3.0)
    slots = g.permutation(pages * PAGE)[:T].astype(np.int64)
    slots[::7] = -1                                              # rows without a slot
    if T > 3:
        slots[3], slots[2] = pages * PAGE, -(1 << 40)            # past the last page, far below the first: skipped
    cache0 = g.integers(0, 256, pages * layers * MX8_PAGE, dtype=np.uint8)
    want = cache0.copy()
    off = (layers - 1) * MX8_PAGE
    put_rows(want, off, layers * MX8_PAGE, slots, rows[:, :ROW])
    cache = to_dev(cache0, dev)
    k3g.call("k3g_latent_mx8_store", to_dev_bf16(rows, dev), stride, to_dev(slots, dev), cache, off, layers * MX8_PAGE, pages, T, k3g.current_stream())
    torch.cuda.synchronize()
    assert np.array_equal(cache.cpu().numpy(), want)             # the rows' bytes, and every other byte as it was


def test_store_extreme_values_as_moe_quant(k3g, dev):
    """Zeros, signed zeros, infinities, NaN, the largest and smallest magnitudes and 448 * 2^k: the bytes k3g_moe_quant
    gives for the same values."""
    import torch
    g = rng(9)
    rows = normal_bf16(g, (64, ROW))
    special = np.array([0x0000, 0x8000, 0x7F80, 0xFF80, 0x7FC0, 0xFFC1, 0x7F7F, 0xFF7F, 0x0001, 0x8001, 0x0080, 0x43E0, 0x43E1, 0x3FE0, 0x3F61], dtype=np.uint16)
    for i in range(32):
        rows[i, :LATENT] = np.where(g.random(LATENT) < 0.1, special[g.integers(0, len(special), LATENT)], rows[i, :LATENT])
    rows[40, :LATENT] = 0
    rows[41, :LATENT] = 0x7FC0
    for i in range(15):
        rows[42 + i, :LATENT] = special[i]
    d = to_dev_bf16(rows, dev)
    cache = torch.zeros(MX8_PAGE, dtype=torch.uint8, device=dev)
    k3g.call("k3g_latent_mx8_store", d, ROW, torch.arange(64, device=dev), cache, 0, MX8_PAGE, 1, 64, k3g.current_stream())
    q = torch.empty((64, LATENT), dtype=torch.uint8, device=dev); sf = torch.empty((64, 16), dtype=torch.uint8, device=dev)
    k3g.call("k3g_moe_quant", d[:, :LATENT].contiguous(), q, sf, 64, LATENT, 0, k3g.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(cache[SCALES_AT:].view(64, 16), sf)
    assert torch.equal(cache[:ROPE_AT].view(64, LATENT), q)
    assert torch.equal(cache[ROPE_AT:SCALES_AT].view(torch.int16).view(64, 64), d[:, LATENT:].contiguous().view(torch.int16))


@pytest.mark.parametrize("n,length", [(1, 1), (1, 0), (63, 64), (65, 64), (64, 63), (700, 513), (130, 1000), (4097, 4097)])
def test_gather(k3g, dev, n, length):
    import torch
    g = rng(n + length)
    width = (n + 63) // 64
    pages, stride = width + 2, 2 * MX8_PAGE
    cache = np.zeros(pages * stride, dtype=np.uint8)
    rows = normal_bf16(g, (64 * pages, ROW), std=5.0)
    put_rows(cache, MX8_PAGE, stride, np.arange(64 * pages), rows)
    table = g.permutation(pages)[:width].astype(np.int32)
    if width > 3:
        table[2], table[3] = -1, pages                           # pages that the cache does not hold
    want, held = mx8_rows(cache, MX8_PAGE, stride, table, n)
    want[min(n, length):] = 0
    out = torch.full((n, ROW), 7.0, dtype=torch.bfloat16, device=dev)
    k3g.call("k3g_latent_mx8_gather", to_dev(cache, dev), to_dev(table, dev), MX8_PAGE, stride, pages, torch.tensor([length], dtype=torch.int32, device=dev), out, n,
             k3g.current_stream())
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().double().numpy(), want)      # exact: bf16 holds code * 2^e


def test_gather_gives_every_code_at_every_scale(k3g, dev):
    """All 256 codes under all 256 scale bytes (NaN codes, the NaN scale, both ends of the exponent range): code * 2^(s - 127)
    rounded once to bf16."""
    import torch
    pages = 16                                                   # 16 scales a row, 1024 rows = 16384 blocks of 32 codes = 8 blocks per scale
    cache = np.zeros((pages, MX8_PAGE), dtype=np.uint8)
    block = np.arange(pages * 64 * 16)
    scale, part = (block // 8 % 256).astype(np.uint8), block % 8
    codes = (part[:, None] * 32 + np.arange(32)[None]).astype(np.uint8)
    cache[:, :ROPE_AT] = codes.reshape(pages, -1)
    cache[:, SCALES_AT:] = scale.reshape(pages, -1)
    out = torch.empty((pages * 64, ROW), dtype=torch.bfloat16, device=dev)
    k3g.call("k3g_latent_mx8_gather", to_dev(cache, dev), torch.arange(pages, dtype=torch.int32, device=dev), 0, MX8_PAGE, pages,
             torch.tensor([pages * 64], dtype=torch.int32, device=dev), out, pages * 64, k3g.current_stream())
    torch.cuda.synchronize()
    want, _ = mx8_rows(cache.reshape(-1), 0, MX8_PAGE, np.arange(pages), pages * 64)
    want = torch.from_numpy(want).float().bfloat16()             # exact in f32; one rounding to bf16
    assert torch.equal(torch.nan_to_num(out.cpu().float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0))


# ---- attention -------------------------------------------------------------------------------------------------------------
class Case:
    """A cache, page tables and queries on the host and on the device."""

    def __init__(self, dev, B, S, heads, prefix, lens, mx8=True, seed=0, layers=2, q_extra=0, scale=192 ** -0.5, q_std=1.4, spare=3, max_pages=None):
        import torch
        g = rng(1000 * seed + B * 100 + S * 10 + heads + prefix)
        self.B, self.S, self.heads, self.scale, self.mx8, self.g, self.dev = B, S, heads, scale, mx8, g, dev
        self.prefix, self.lens = prefix, np.asarray(lens, dtype=np.int32)
        self.max_pages = max_pages if max_pages is not None else max(1, max((int(n) + 63) // 64 for n in lens))
        self.prefix_pages = (prefix + 63) // 64
        need = self.prefix_pages + B * self.max_pages
        self.pages = need + spare
        order = g.permutation(self.pages).astype(np.int32)
        self.prefix_table, self.tables = order[:self.prefix_pages].copy(), order[self.prefix_pages:need].reshape(B, self.max_pages).copy()
        rows = normal_bf16(g, (self.pages * 64, ROW))
        if mx8:
            self.page, self.off, self.stride = MX8_PAGE, (layers - 1) * MX8_PAGE, layers * MX8_PAGE
            self.cache = np.zeros(self.pages * self.stride, dtype=np.uint8)
            q, rope, sf = quant_rows(rows)
            c = self.cache.reshape(self.pages, self.stride)[:, self.off:self.off + MX8_PAGE]
            c[:, :ROPE_AT] = q.reshape(self.pages, -1)
            c[:, ROPE_AT:SCALES_AT] = np.ascontiguousarray(rope).view(np.uint8).reshape(self.pages, -1)
            c[:, SCALES_AT:] = sf.reshape(self.pages, -1)
        else:
            self.page, self.off, self.stride = PAGE * ROW, (layers - 1) * PAGE * ROW, layers * PAGE * ROW
            self.cache = np.zeros(self.pages * self.stride, dtype=np.uint16)
            self.cache.reshape(self.pages, self.stride)[:, self.off:self.off + self.page] = rows.reshape(self.pages, -1)
        self.q = normal_bf16(g, (B, S, heads * ROW + q_extra), std=q_std)
        self.out0 = normal_bf16(g, (B, S, heads, LATENT))

    def set_token(self, table, t, values):
        """Overwrite token t of a table with 576 bf16 bit patterns."""
        pid = int(table[t // 64])
        if self.mx8:
            put_rows(self.cache, self.off, self.stride, [pid * 64 + t % 64], values.reshape(1, ROW))
        else:
            o = pid * self.stride + self.off + (t % 64) * ROW
            self.cache[o:o + ROW] = values

    def upload(self, k3g):
        import torch
        d = self.dev
        up = lambda a: to_dev(a, d)
        self.d_cache = up(self.cache) if self.mx8 else to_dev_bf16(self.cache, d)
        self.d_q, self.d_lens, self.d_tables = to_dev_bf16(self.q, d), up(self.lens), up(self.tables)
        self.d_pt = up(self.prefix_table) if self.prefix_pages else None
        self.d_pl = torch.tensor([self.prefix], dtype=torch.int32, device=d)
        self.out = to_dev_bf16(self.out0, d)
        self.ws = torch.empty(k3g.latent_attn_workspace(self.B, self.S, self.heads), dtype=torch.uint8, device=d)
        return self

    def call(self, k3g, out=None, ws=None):
        out, ws = self.out if out is None else out, self.ws if ws is None else ws
        k3g.call("k3g_latent_attn", self.d_q, self.q.shape[2], self.d_cache, int(self.mx8), self.off, self.stride, self.pages, self.d_pt, self.d_pl,
                 self.prefix_pages, self.d_tables, self.d_lens, self.max_pages, out, ws, ws.numel(), self.B, self.S, self.heads, self.scale,
                 k3g.current_stream())

    def oracle(self):
        read = mx8_rows if self.mx8 else bf16_rows
        q = k3o.bf16_to_f32(np.ascontiguousarray(self.q[:, :, :self.heads * ROW])).astype(np.float64).reshape(self.B, self.S, self.heads, ROW)
        return attn_oracle(q, lambda t, n: read(self.cache, self.off, self.stride, t, n), self.prefix_table, self.prefix, self.tables, self.lens, self.scale)

    def check(self, k3g):
        import torch
        self.upload(k3g).call(k3g)
        torch.cuda.synchronize()
        self.compare(bf16_bits(self.out))

    def compare(self, bits):
        want, spread, ds = self.oracle()
        got = k3o.bf16_to_f32(bits).astype(np.float64)
        live = self.lens >= 0
        assert np.array_equal(bits[~live], self.out0[~live])     # rows of no sequence are left as they were
        want, got, spread, ds = want[live], got[live], spread[live], ds[live]
        assert int((np.isnan(got) != np.isnan(want)).sum()) == 0
        fin = np.isfinite(want)
        off = np.abs(got - np.where(fin, want, 0)) - attn_tolerance(np.where(fin, want, 0), spread, ds)
        assert np.all(off[fin] <= 0), "worst excess %g" % off[fin].max()


@pytest.mark.parametrize("mx8", [True, False])
@pytest.mark.parametrize("B,S,heads,prefix,lens", [
    (1, 1, 1, 0, [1]), (1, 1, 24, 0, [64]), (1, 1, 24, 64, [0]), (2, 1, 12, 1, [65, 1]), (3, 2, 5, 63, [2, 128, 1]), (2, 3, 24, 65, [3, 200]),
    (5, 4, 24, 129, [4, 64, 65, 67, 130]), (1, 1, 96, 1000, [100]), (2, 7, 16, 0, [7, 70]), (1, 5, 48, 200, [1]), (40, 1, 3, 300, list(range(40))),
    (7, 1, 65, 640, [0, 1, 63, 64, 65, 127, 128]), (2, 2, 64, 0, [300, 500])])
def test_attn(k3g, dev, mx8, B, S, heads, prefix, lens):
    Case(dev, B, S, heads, prefix, lens, mx8=mx8, seed=1).check(k3g)


@pytest.mark.parametrize("mx8", [True, False])
def test_attn_many_tokens_split_over_the_card(k3g, dev, mx8):
    """Few rows and a long prefix: the tokens are split over all SMs and joined."""
    Case(dev, 2, 1, 24, 20000, [70, 3], mx8=mx8, seed=2).check(k3g)


@pytest.mark.parametrize("mx8", [True, False])
@pytest.mark.parametrize("B,S,heads", [(50, 3, 9), (101, 5, 5), (49, 1, 24)])
def test_attn_rows_joined_by_one_two_and_four_teams(k3g, dev, mx8, B, S, heads):
    """Row counts on either side of the join's borders, and sequences whose rows do not begin at multiples of four."""
    Case(dev, B, S, heads, 1000, [S + (i * 29) % 150 for i in range(B)], mx8=mx8, seed=31).check(k3g)


@pytest.mark.parametrize("B", [148, 149])
def test_attn_rows_on_either_side_of_one_team(k3g, dev, B):
    Case(dev, B, 1, 24, 130, [1 + (i * 29) % 150 for i in range(B)], seed=35).check(k3g)


def test_attn_many_rows(k3g, dev):
    """More row tiles than SMs, with sequences that begin inside a tile."""
    Case(dev, 150, 3, 24, 130, [3 + (i * 37) % 100 for i in range(150)], seed=3).check(k3g)


def test_attn_large_scores_and_negative_scale(k3g, dev):
    """Scores of +-60: the running maximum moves by more than the exponent's range can hold unscaled.  The second case turns the order round."""
    for scale in (0.06, -0.06):
        Case(dev, 2, 2, 24, 700, [300, 90], seed=4, scale=scale, q_std=20.0, mx8=False).check(k3g)


def test_attn_scores_that_grow_token_by_token(k3g, dev):
    """Every page raises the maximum by about 20 (base e): what was summed before has to be scaled down again and again."""
    c = Case(dev, 1, 1, 24, 64 * 12, [64], seed=5, mx8=False, scale=1.0, q_std=0.0)
    c.q[..., :] = 0
    c.q.reshape(1, 1, 24, ROW)[..., 575] = 0x3F80               # q = 1 on the last rope column: the score is that column of the key
    for t in range(64 * 12):
        pid = int(c.prefix_table[t // 64])
        c.cache[pid * c.stride + c.off + (t % 64) * ROW + 575] = k3o.f32_to_bf16(np.float32([20.0 * (t // 64) + 0.25 * (t % 7) - 100]))[0]
    c.check(k3g)


@pytest.mark.parametrize("mx8", [True, False])
def test_attn_lengths_that_leave_rows_empty(k3g, dev, mx8):
    """No prefix: sequences with no token, with fewer tokens than steps (the first steps see nothing), and padded ones."""
    Case(dev, 5, 4, 24, 0, [0, 2, -1, 4, -7], mx8=mx8, seed=6).check(k3g)
    Case(dev, 3, 2, 24, 10, [-1, -1, -1], mx8=mx8, seed=7, max_pages=1).check(k3g)


@pytest.mark.parametrize("mx8", [True, False])
def test_attn_no_own_tokens_at_all_and_null_tables(k3g, dev, mx8):
    c = Case(dev, 3, 1, 24, 100, [0, 0, 0], mx8=mx8, seed=8, max_pages=0)
    c.check(k3g)
    c = Case(dev, 2, 1, 24, 0, [0, 0], mx8=mx8, seed=8, max_pages=0)
    c.check(k3g)                                                 # nothing anywhere: zeros


@pytest.mark.parametrize("mx8", [True, False])
def test_attn_garbage_behind_the_last_token_and_beside_the_tables(k3g, dev, mx8):
    """NaN and infinities in every cache byte that no length reaches: the rest of the last pages, unused pages, the other
    layer, table entries behind the last page that lie outside the cache."""
    c = Case(dev, 4, 3, 24, 70, [3, 64, 65, 100], mx8=mx8, seed=9, max_pages=4)
    g, seen = rng(10), set()
    for t in range(c.prefix):
        seen.add((int(c.prefix_table[t // 64]), t % 64))
    for b in range(c.B):
        for t in range(int(c.lens[b])):
            seen.add((int(c.tables[b, t // 64]), t % 64))
        c.tables[b, (int(c.lens[b]) + 63) // 64:] = [1 << 30, -5, c.pages][:c.max_pages - (int(c.lens[b]) + 63) // 64]
    full = c.cache.reshape(c.pages, c.stride)
    keep = full.copy()
    if mx8:
        full[:] = 0xFF
        full[:, c.off + ROPE_AT:c.off + SCALES_AT:2] = 0x80      # bf16 0x7f80: infinity
        full[:, c.off + ROPE_AT + 1:c.off + SCALES_AT:2] = 0x7F
    else:
        full[:] = 0x7F80
        full[:, ::3] = 0x7FC0
    for p, r in seen:
        if mx8:
            for lo, n in ((r * LATENT, LATENT), (ROPE_AT + r * 128, 128), (SCALES_AT + r * 16, 16)):
                full[p, c.off + lo:c.off + lo + n] = keep[p, c.off + lo:c.off + lo + n]
        else:
            full[p, c.off + r * ROW:c.off + (r + 1) * ROW] = keep[p, c.off + r * ROW:c.off + (r + 1) * ROW]
    c.check(k3g)


@pytest.mark.parametrize("mx8", [True, False])
@pytest.mark.parametrize("bad", [0x7FC0, 0x7F80])
def test_attn_a_bad_token_reaches_the_rows_that_see_it_and_no_others(k3g, dev, mx8, bad):
    """A NaN (or an infinity in the rope columns) in a drafted token's latent: that step and the later ones are NaN, the earlier
    steps and the other sequences are as if it was not there.  Then one in the prefix: everything is NaN."""
    g = rng(11)
    c = Case(dev, 3, 4, 24, 40, [66, 66, 10], mx8=mx8, seed=11)
    v = normal_bf16(g, (ROW,))
    v[530 if bad == 0x7F80 else 17] = bad
    c.set_token(c.tables[1], 64, v)                              # seen by steps 2 and 3 of sequence 1
    c.check(k3g)
    want, _, _ = c.oracle()
    assert np.isnan(want[1, 2:]).all() and np.isfinite(want[1, :2]).all() and np.isfinite(want[0]).all()
    if bad == 0x7FC0:
        c = Case(dev, 2, 2, 5, 40, [66, 2], mx8=mx8, seed=12)
        c.set_token(c.prefix_table, 7, v)
        c.check(k3g)


@pytest.mark.parametrize("mx8", [True, False])
def test_attn_pages_that_the_cache_does_not_hold_are_not_read(k3g, dev, mx8):
    c = Case(dev, 2, 1, 24, 200, [130, 64], mx8=mx8, seed=13)
    c.prefix_table[1], c.tables[0, 0], c.tables[1, 0] = -1, c.pages, 1 << 30
    c.check(k3g)


def test_attn_lengths_beyond_the_tables_are_cut(k3g, dev):
    import torch
    c = Case(dev, 2, 2, 24, 128, [128, 64], seed=14)
    c.prefix, c.lens = 1 << 30, np.array([2 ** 31 - 1, 64], dtype=np.int32)
    c.check(k3g)


def test_attn_strided_queries(k3g, dev):
    Case(dev, 3, 2, 24, 100, [5, 70, 64], seed=15, q_extra=128).check(k3g)


def test_attn_page_offsets_beyond_32_bits(k3g, dev):
    """Pages 1.5 GB apart: the third begins behind 2^31 bytes, the fourth behind 2^32."""
    import torch
    c = Case(dev, 1, 1, 24, 0, [4 * 64 - 3], seed=16, layers=1, spare=0)
    c.tables[0] = [3, 1, 0, 2]
    want = c.oracle()
    c.upload(k3g)
    stride = 3 << 29
    big = torch.empty(3 * stride + MX8_PAGE, dtype=torch.uint8, device=dev)
    for p in range(4):
        big[p * stride:p * stride + MX8_PAGE] = c.d_cache[p * MX8_PAGE:(p + 1) * MX8_PAGE]
    c.call(k3g)
    torch.cuda.synchronize()
    near = bf16_bits(c.out)
    c.compare(near)
    c.d_cache, c.stride = big, stride
    c.out.zero_()
    c.call(k3g)
    torch.cuda.synchronize()
    assert np.array_equal(bf16_bits(c.out), near)
    # the same pages read back and written where they lie
    back = torch.empty((4 * 64, ROW), dtype=torch.bfloat16, device=dev)
    k3g.call("k3g_latent_mx8_gather", big, c.d_tables, 0, stride, 4, torch.tensor([256], dtype=torch.int32, device=dev), back, 256, k3g.current_stream())
    slots = (c.d_tables.long().view(4, 1) * 64 + torch.arange(64, device=dev)).view(-1)
    for p in range(4):
        big[p * stride:p * stride + MX8_PAGE] = 0
    k3g.call("k3g_latent_mx8_store", back, ROW, slots, big, 0, stride, 4, 256, k3g.current_stream())
    torch.cuda.synchronize()
    again = torch.empty_like(back)
    k3g.call("k3g_latent_mx8_gather", big, c.d_tables, 0, stride, 4, torch.tensor([256], dtype=torch.int32, device=dev), again, 256, k3g.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), back.view(torch.int16))


def test_attn_same_bits_every_time_and_on_two_streams_at_once(k3g, dev):
    import torch
    c = Case(dev, 9, 2, 24, 3000, [10 + 50 * i for i in range(9)], seed=17).upload(k3g)
    c.call(k3g)
    torch.cuda.synchronize()
    first = c.out.clone()
    c.ws.random_(0, 256)                                         # what a workspace holds beforehand does not matter
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(c.out) for _ in range(2)]
    spaces = [c.ws, torch.randint(0, 256, c.ws.shape, dtype=torch.uint8, device=dev)]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, o, w in zip(streams, outs, spaces):
            with torch.cuda.stream(st):
                c.call(k3g, out=o, ws=w)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.view(torch.int16), first.view(torch.int16))


def test_attn_captured_once_serves_growing_lengths(k3g, dev):
    """One graph, replayed while the sequences grow across page borders, one ends and the prefix is exchanged: lengths and
    tables are read on the device at every replay."""
    import torch
    c = Case(dev, 3, 2, 24, 150, [60, 2, 127], seed=18, max_pages=3).upload(k3g)
    c.call(k3g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.call(k3g)
    for step in range(6):
        c.lens = np.array([60 + 2 * step, 2 + 30 * step, -1 if step == 4 else 127 + step], dtype=np.int32)
        c.prefix = [150, 150, 128, 0, 64, 150][step]
        c.d_lens.copy_(torch.from_numpy(c.lens)); c.d_pl.fill_(c.prefix)
        c.out.copy_(to_dev_bf16(c.out0, dev))
        graph.replay()
        torch.cuda.synchronize()
        c.compare(bf16_bits(c.out))


@pytest.mark.parametrize("mx8", [True, False])
def test_attn_stretches_of_one_tile_one_after_another(k3g, dev, mx8):
    """Hundreds of sequences that fit one tile: every CTA takes several stretches of a single tile, in which the exchange of the row maxima is
    followed at once by that of the sums through the same words.  The oracle's results, and the same bits in thirty runs."""
    import torch
    c = Case(dev, 600, 1, 24, 0, [1 + (i * 53) % 128 for i in range(600)], mx8=mx8, seed=33, layers=1).upload(k3g)
    c.call(k3g)
    torch.cuda.synchronize()
    c.compare(bf16_bits(c.out))
    first = c.out.clone()
    for _ in range(30):
        c.out.zero_()
        c.call(k3g)
        assert torch.equal(c.out.view(torch.int16), first.view(torch.int16))


def test_attn_workspace_at_any_16_bytes(k3g, dev):
    """Only 16-byte aligned, and exactly as large as asked for: what lies around it stays."""
    import torch
    c = Case(dev, 3, 2, 24, 700, [5, 70, 3], seed=32).upload(k3g)
    n = c.ws.numel()
    buf = torch.full((n + 64,), 0xA5, dtype=torch.uint8, device=dev)
    for off in (0, 16, 32, 48):
        buf.fill_(0xA5)
        c.out.copy_(to_dev_bf16(c.out0, dev))
        c.call(k3g, ws=buf[off:off + n])
        torch.cuda.synchronize()
        c.compare(bf16_bits(c.out))
        assert (buf[:off] == 0xA5).all() and (buf[off + n:] == 0xA5).all()


def test_attn_workspace_of_a_larger_batch_serves_a_smaller_one(k3g, dev):
    import torch
    big = k3g.latent_attn_workspace(8, 4, 96)
    c = Case(dev, 2, 1, 24, 100, [5, 70], seed=19).upload(k3g)
    assert big >= c.ws.numel()
    c.ws = torch.full((big,), 0xFF, dtype=torch.uint8, device=dev)
    c.call(k3g)
    torch.cuda.synchronize()
    c.compare(bf16_bits(c.out))


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("bad", [0x7F80, 0xFF80])
def test_attn_an_infinite_latent_that_every_step_sees(k3g, dev, own, bad):
    """An infinity in a latent column, on bf16 pages, in the prefix or among the tokens of a batch without drafts: rows whose score of that token is
    +infinity are NaN, for the others it weighs nothing, but 0 times the infinity makes that column of their outputs NaN.  Other sequences
    do not see an own token."""
    import torch
    c = Case(dev, 2, 1, 24, 100, [70, 30], mx8=False, seed=80 + own, max_pages=2)
    table, t = (c.tables[0], 33) if own else (c.prefix_table, 77)
    at = int(table[t // 64]) * c.stride + c.off + (t % 64) * ROW
    c.cache[at + 17] = bad
    c.upload(k3g).call(k3g)
    torch.cuda.synchronize()
    got = k3o.bf16_to_f32(bf16_bits(c.out)).astype(np.float64)
    q17 = k3o.bf16_to_f32(np.ascontiguousarray(c.q)).reshape(c.B, c.S, c.heads, ROW)[..., 17]
    up = (q17 > 0) == (bad == 0x7F80)
    seen = np.array([True, not own])[:, None, None]
    assert (q17 != 0).all() and (up & seen).any() and (~up & seen).any()
    read = lambda tab, n: _rows_but(c, tab, n, int(table[t // 64]), t % 64)
    q = k3o.bf16_to_f32(np.ascontiguousarray(c.q)).astype(np.float64).reshape(c.B, c.S, c.heads, ROW)
    want, spread, ds = attn_oracle(q, read, c.prefix_table, c.prefix, c.tables, c.lens, c.scale)
    nan = np.isnan(got)
    assert nan[up & seen].all()
    assert np.array_equal(nan[~up & seen], np.broadcast_to(np.arange(LATENT) == 17, nan[~up & seen].shape)) and not nan[~(up & seen) & ~seen].any()
    off = np.abs(np.where(nan, want, got) - want) - attn_tolerance(want, spread, ds)
    assert np.all(off <= 0)


def _rows_but(c, table, n, page, at):
    rows, held = bf16_rows(c.cache, c.off, c.stride, table, n)
    for t in range(at, n, 64):
        if int(table[t // 64]) == page:
            rows[t], held[t] = 0, False
    return rows, held


# ---- exponents of MXFP8 pages ------------------------------------------------------------------------------------------------
def _fill(c, rows):
    """The whole cache of an MXFP8 case from rows [pages * 64, 576] of floats."""
    c.rows = rows
    q, rope, sf = quant_rows(k3o.f32_to_bf16(rows.astype(np.float32).reshape(-1)).reshape(rows.shape))
    at = c.cache.reshape(c.pages, c.stride)[:, c.off:c.off + MX8_PAGE]
    at[:, :ROPE_AT] = q.reshape(c.pages, -1)
    at[:, ROPE_AT:SCALES_AT] = np.ascontiguousarray(rope).view(np.uint8).reshape(c.pages, -1)
    at[:, SCALES_AT:] = sf.reshape(c.pages, -1)
    return c


def _token(table, t):
    return int(table[t // 64]) * 64 + t % 64


@pytest.mark.parametrize("where", ["row beside", "block beside", "sixteen rows", "rows of another tile", "every other row"])
@pytest.mark.parametrize("size", [-10, -20, -30])
def test_attn_mx8_zeros_beside_small_latents(k3g, dev, size, where):
    """A block of zeros has scale byte 127 whatever lies beside it: it takes nothing from the range of the tokens that are not zero."""
    c = Case(dev, 2, 2, 12, 300, [70, 200], seed=40 - size)
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    rows[:, :LATENT] *= 2.0 ** size
    p = c.prefix_table
    if where == "row beside":
        rows[[_token(p, 5), _token(c.tables[0], 66), _token(c.tables[1], 199)], :LATENT] = 0
    elif where == "block beside":
        rows[[_token(p, t) for t in range(3, 300, 16)], 64:96] = 0
        rows[_token(c.tables[1], 130), 480:512] = -0.0
    elif where == "sixteen rows":
        rows[[_token(p, t) for t in range(16, 32)], :LATENT] = 0
    elif where == "rows of another tile":
        rows[[_token(p, t) for t in range(256, 300)], :LATENT] = 0
        rows[[_token(c.tables[1], t) for t in range(128)], :LATENT] = -0.0
    else:
        rows[::2, :LATENT] = 0
    _fill(c, rows).check(k3g)


@pytest.mark.parametrize("where", ["sixteen rows", "rows of another tile", "the first tiles", "all but a few", "all"])
@pytest.mark.parametrize("size", [0, 40, 60, 115])
def test_attn_mx8_zeros_beside_large_latents(k3g, dev, size, where):
    """Tokens that are all zeros weigh what their scores give, however large the others' latents are, and whether they come first or last."""
    c = Case(dev, 2, 2, 12, 700, [70, 200], seed=46 + size)
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    rows[:, :LATENT] *= np.float32(2.0 ** size)
    p = c.prefix_table
    if where == "sixteen rows":
        rows[[_token(p, t) for t in range(16, 32)], :LATENT] = 0
    elif where == "rows of another tile":
        rows[[_token(p, t) for t in range(256, 600)], :LATENT] = 0
        rows[[_token(c.tables[1], t) for t in range(128)], :LATENT] = -0.0
    elif where == "the first tiles":
        rows[[_token(p, t) for t in range(690)], :LATENT] = 0
    elif where == "all but a few":
        keep = [_token(p, 450), _token(c.tables[0], 20), _token(c.tables[1], 180)]
        rows[np.setdiff1d(np.arange(len(rows)), keep), :LATENT] = 0
    else:
        rows[:, :LATENT] = 0
    _scale_q(c, [2.0 ** -size] * c.heads)
    _check_range(_fill(c, rows), k3g)


@pytest.mark.parametrize("zeros", [False, True])
def test_attn_mx8_a_nan_scale_over_codes_of_zero(k3g, dev, zeros):
    """Scale byte 255 is NaN whatever it scales, with a block of zeros among the sixteen tokens and without."""
    c = Case(dev, 2, 1, 12, 0, [70, 30], seed=45)
    t = _token(c.tables[0], 20)
    if zeros:
        c.set_token(c.tables[0], 19, np.zeros(ROW, dtype=np.uint16))
    page = c.cache.reshape(c.pages, c.stride)[t // 64, c.off:]
    page[t % 64 * LATENT + 96:t % 64 * LATENT + 128] = 0
    page[SCALES_AT + t % 64 * 16 + 3] = 255
    c.check(k3g)
    want, _, _ = c.oracle()
    assert np.isnan(want[0]).all() and np.isfinite(want[1]).all()


def _scale_q(c, heads):
    """Latent columns of the queries times a factor for each head (powers of two, or 0)."""
    f = k3o.bf16_to_f32(np.ascontiguousarray(c.q)).reshape(c.B, c.S, c.heads, ROW)
    f[..., :LATENT] *= np.asarray(heads, dtype=np.float32).reshape(-1, 1)
    c.q = k3o.f32_to_bf16(f.reshape(-1)).reshape(c.q.shape)


def _check_range(c, k3g):
    """As Case.check, with what f16 operands may lose beside it."""
    import torch
    c.upload(k3g).call(k3g)
    torch.cuda.synchronize()
    got = k3o.bf16_to_f32(bf16_bits(c.out)).astype(np.float64)
    want, spread, ds = c.oracle()
    q = k3o.bf16_to_f32(np.ascontiguousarray(c.q)).astype(np.float64).reshape(c.B, c.S, c.heads, ROW)
    lost, dlost = mx8_range_tolerance(q, lambda t, n: mx8_rows(c.cache, c.off, c.stride, t, n), c.prefix_table, c.prefix, c.tables, c.lens, c.scale)
    off = np.abs(got - want) - attn_tolerance(want, spread, ds) - 3 * dlost[..., None] * spread - lost[..., None]
    assert np.all(off <= 0), "worst excess %g" % off.max()


@pytest.mark.parametrize("scale", [0.07, -0.07])
@pytest.mark.parametrize("kind", ["blocks", "blocks upwards", "tokens", "tiles", "pages of 2^-30", "tiles of 2^20"])
def test_attn_mx8_magnitudes_that_differ(k3g, dev, kind, scale):
    """Scales that spread over 2^30 and more within a token, within 16 tokens and from tile to tile."""
    c = Case(dev, 2, 2, 12, 700, [70, 200], seed=50, scale=scale)
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    token, block = np.arange(c.pages * 64)[:, None], np.arange(LATENT)[None] // 32
    if kind == "blocks":
        up = -np.round(2.2 * block) + 0 * token                  # 0 .. -33
    elif kind == "blocks upwards":
        up = np.round(1.4 * block) - 20 + token % 3 - 1          # the last block largest
    elif kind == "tokens":
        up = (token * 7 % 16) * -2 + 0 * block                   # 0 .. -30
    elif kind == "tiles":
        up = c.g.integers(-20, 21, c.pages)[token // 64] + 0 * block
    elif kind == "pages of 2^-30":
        up = np.where(token // 64 % 2 == 0, -30, 0) + 0 * block
    else:
        up = np.where(token // 128 % 3 == 1, 20, 0) + 0 * block
    rows[:, :LATENT] *= 2.0 ** up
    rows[::37, :LATENT] = 0
    _scale_q(c, [2.0 ** -max(0, int(up.max()))] * c.heads)
    _check_range(_fill(c, rows), k3g)


@pytest.mark.parametrize("size", [-90, -75, 60, 115])
def test_attn_mx8_latents_at_the_ends_of_the_exponents(k3g, dev, size):
    """Latents of 2^-90 (where E has reached its least) to 2^115, queries that make scores of ordinary size of them, zeros among them."""
    c = Case(dev, 2, 2, 12, 150, [70, 130], seed=55, scale=0.07)
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    rows[:, :LATENT] *= np.float32(2.0 ** size)
    rows[::23, :LATENT] = 0
    _scale_q(c, [2.0 ** -size] * c.heads)
    _check_range(_fill(c, rows), k3g)


@pytest.mark.parametrize("scale", [0.07, -0.07])
@pytest.mark.parametrize("size", [-40, 0, 12])
def test_attn_mx8_query_rows_of_any_size(k3g, dev, size, scale):
    """Queries from 2^-40 to 2^40 beside one another, rows of zeros among them, so that scores count at one end."""
    c = Case(dev, 3, 2, 11, 260, [5, 70, 128], seed=60 + size, scale=scale)
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    rows[:, :LATENT] *= 2.0 ** size
    heads = [2.0 ** (10 * h - 40) if 10 * h - 40 <= -size else 0.0 for h in range(9)] + [0.0, 2.0 ** -size]
    _scale_q(c, heads)
    c.q.reshape(c.B, c.S, c.heads, ROW)[:, 0, 9] = 0             # zeros in the rope columns, too
    c.q.reshape(c.B, c.S, c.heads, ROW)[1, 1] = 0
    _check_range(_fill(c, rows), k3g)


def test_attn_mx8_queries_below_the_normal_numbers(k3g, dev):
    """Query rows of subnormal bf16 against latents of 2^110: their scores are ordinary ones, with a scale of 2^15."""
    c = Case(dev, 2, 1, 6, 100, [70, 130], seed=75, scale=2.0 ** 15)
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    rows[:, :LATENT] *= np.float32(2.0 ** 110)
    q = c.g.integers(0, 64, c.q.shape).astype(np.uint16) | (c.g.integers(0, 2, c.q.shape) << 15).astype(np.uint16)   # up to 2^-127
    q.reshape(c.B, c.S, c.heads, ROW)[..., LATENT:] = 0
    c.q = q
    _check_range(_fill(c, rows), k3g)


@pytest.mark.parametrize("scale", [0.06, -0.06])
def test_attn_mx8_large_scores(k3g, dev, scale):
    """As with bf16 pages: scores of +-60, and the order turned round."""
    Case(dev, 2, 2, 24, 700, [300, 90], seed=4, scale=scale, q_std=20.0).check(k3g)


@pytest.mark.parametrize("jump", [0, 20])
@pytest.mark.parametrize("sign", [1, -1])
def test_attn_mx8_scores_that_grow_token_by_token(k3g, dev, sign, jump):
    """Every page raises the maximum by about 20 (base e), with latents of one size or of sizes that change by 2^20 from page to page: what was
    summed before is scaled down again and again, in units that the exponents shift."""
    c = Case(dev, 1, 1, 24, 64 * 12, [64], seed=70, scale=float(sign), q_std=0.0)
    c.q[..., :] = 0
    c.q.reshape(1, 1, 24, ROW)[..., 575] = 0x3F80               # q = 1 on the last rope column: the score is that column of the key
    rows = normal_bf16(c.g, (c.pages * 64, ROW))
    rows = k3o.bf16_to_f32(rows.reshape(-1)).reshape(rows.shape).copy()
    for t in range(64 * 12):
        rows[_token(c.prefix_table, t), 575] = sign * (20.0 * (t // 64) + 0.25 * (t % 7) - 100)
        rows[_token(c.prefix_table, t), :LATENT] *= 2.0 ** (jump * (t // 64 % 2))
    _check_range(_fill(c, rows), k3g)


# ---- verification ------------------------------------------------------------------------------------------------------------
def _probs(g, shape, std=2.5):
    x = g.standard_normal(shape) * std
    x = np.exp(x - x.max(-1, keepdims=True))
    return (x / x.sum(-1, keepdims=True)).astype(np.float32)


def _verify(k3g, dev, target, draft, ids, u, stride=None):
    import torch
    B, S = ids.shape
    V = target.shape[2]
    st = stride or V
    pad = lambda a: np.concatenate([a, np.full(a.shape[:2] + (st - V,), 9.0, dtype=np.float32)], 2)      # what lies between the rows is not probability
    acc = torch.full((B + 1,), 77, dtype=torch.int32, device=dev); tok = torch.full((B + 1, S + 1), 77, dtype=torch.int64, device=dev)
    k3g.call("k3g_verify_draft", to_dev(pad(target), dev), st, None if draft is None else to_dev(pad(draft), dev), st, to_dev(ids.astype(np.int64), dev) if S else tok, to_dev(u, dev),
             acc, tok, B, S, V, k3g.current_stream())
    torch.cuda.synchronize()
    assert acc[B] == 77 and (tok[B] == 77).all()                 # nothing behind the last sequence
    return acc[:B].cpu().numpy(), tok[:B].cpu().numpy()


@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("B,S,V,stride", [(1, 1, 1, None), (1, 3, 5, None), (3, 4, 129, None), (9, 2, 2048, None), (5, 5, 4099, None), (4, 8, 32000, 32004), (2, 32, 1000, None),
                                          (700, 1, 257, 260), (80, 3, 20000, None), (2, 3, 163840, None), (3, 0, 500, None), (1, 2, 500001, None)])
def test_verify(k3g, dev, with_probs, B, S, V, stride):
    g = rng(B + S + V)
    target = _probs(g, (B, S + 1, V))
    draft = _probs(g, (B, S, V)) if with_probs else None
    ids = np.argmax(target[:, :S], -1) if not with_probs else g.integers(0, V, (B, S))
    if with_probs and S:
        near = (g.random((B, S)) < 0.8)[..., None]               # most drafts come from a model close to the target
        draft = np.where(near, target[:, :S] * np.float32(0.9) + draft * np.float32(0.1), draft).astype(np.float32)
        ids = np.where(near[..., 0], np.argmax(target[:, :S], -1), ids)
    u = g.random((B, S + 1), dtype=np.float32)
    acc, tok = _verify(k3g, dev, target, draft, ids, u, stride)
    o_acc, o_tok = verify_oracle(target, draft, ids, u)
    assert np.array_equal(acc, o_acc) and np.array_equal(tok, o_tok)


@pytest.mark.parametrize("B,V", [(74, 4095), (74, 4096), (75, 32767), (75, 32768), (80, 131072), (19, 131071)])
def test_verify_blocks_per_sequence(k3g, dev, B, V):
    """On either side of the borders between one, two, four and eight blocks a sequence, and with more clusters than the card holds at once."""
    g = rng(B + V)
    target, draft = _probs(g, (B, 2, V)), _probs(g, (B, 1, V))
    ids, u = g.integers(0, V, (B, 1)), g.random((B, 2), dtype=np.float32)
    ids[::2, 0] = np.argmax(target[::2, 0], -1)
    acc, tok = _verify(k3g, dev, target, draft, ids, u)
    o_acc, o_tok = verify_oracle(target, draft, ids, u)
    assert 0 < o_acc.sum() < B and np.array_equal(acc, o_acc) and np.array_equal(tok, o_tok)


def test_verify_borders(k3g, dev):
    """Exact ties, both ends of the random numbers, drafts of probability 0, equal distributions, empty and spoilt rows."""
    V = 8
    half = np.array([0.5, 0.25, 0.125, 0.125, 0, 0, 0, 0], dtype=np.float32)
    last = np.array([0, 0, 0, 0, 0, 0, 0.25, 0.75], dtype=np.float32)
    none = np.zeros(V, dtype=np.float32)
    spoilt = np.array([np.nan, -1, np.inf, 0.5, -np.inf, 0.5, 0, 0], dtype=np.float32)
    top = np.nextafter(np.float32(1), np.float32(0))
    cases = []
    for p0, p1 in ((half, last), (last, half), (none, none), (spoilt, spoilt), (half, none), (half, spoilt)):
        for q0 in (half, last, none, spoilt):
            for x in (0, 3, 4, 7, -1, 8, 1 << 40):
                for u0 in (0.0, 0.25, 0.5, top):
                    for u1 in (0.0, 0.25, 0.5, 0.875, top):
                        cases.append((p0, p1, q0, x, u0, u1))
    target = np.stack([np.stack([c[0], c[1]]) for c in cases]); draft = np.stack([c[2][None] for c in cases])
    ids = np.array([[c[3]] for c in cases], dtype=np.int64); u = np.array([[c[4], c[5]] for c in cases], dtype=np.float32)
    for d in (draft, None):
        acc, tok = _verify(k3g, dev, target, d, ids, u)
        o_acc, o_tok = verify_oracle(target, d, ids, u)
        assert np.array_equal(acc, o_acc) and np.array_equal(tok, o_tok)


def test_verify_random_number_of_one_takes_the_last_token_with_a_weight(k3g, dev):
    g = rng(21)
    target = _probs(g, (2, 1, 5000)); target[:, :, 4900:] = 0
    acc, tok = _verify(k3g, dev, target, None, np.zeros((2, 0), dtype=np.int64), np.array([[1.0], [np.nan]], dtype=np.float32))
    assert (acc == 0).all() and (tok[:, 0] == 4899).all()


# ---- together ------------------------------------------------------------------------------------------------------------------
def test_decode_steps_with_drafts_over_one_prompt(k3g, dev):
    """The operators as a decoding program runs them: the prompt's latents appended by k3g_mla_prep to bf16 pages, quantised into MXFP8 pages and read
    back; then steps of a batch that shares the prompt, captured into one graph: three latents per sequence appended, attention,
    a small output head, verification of two drafts.  The attention's rows are compared with the oracle, the tokens with the oracle on
    the kernel's own probabilities, at every step; sequences grow by what was accepted, across a page border."""
    import torch
    g = rng(30)
    tg = torch.Generator(device=dev); tg.manual_seed(30)
    B, S, heads, V, prompt, max_pages, steps = 4, 3, 6, 1000, 150, 2, 5
    pp = (prompt + 63) // 64
    pages = pp + B * max_pages
    partial = normal_bf16(g, (prompt, 2112))
    gq, gkv = normal_bf16(g, (1536,), mean=1.0, std=0.02), normal_bf16(g, (512,), mean=1.0, std=0.02)
    slab = torch.zeros(pp * 64 * ROW, dtype=torch.bfloat16, device=dev)
    qn = torch.empty((prompt, 1536), dtype=torch.bfloat16, device=dev)
    slots = torch.arange(prompt, device=dev)
    s = k3g.current_stream
    k3g.call("k3g_mla_prep", to_dev_bf16(partial, dev), 1, to_dev_bf16(gq, dev), to_dev_bf16(gkv, dev), slots, slab, 0, 64 * ROW, qn, None, prompt, 0, 1e-5, s())
    cache = torch.zeros(pages * MX8_PAGE, dtype=torch.uint8, device=dev)
    k3g.call("k3g_latent_mx8_store", slab, ROW, slots, cache, 0, MX8_PAGE, pages, prompt, s())
    prefix_table = torch.arange(pp, dtype=torch.int32, device=dev)
    plen = torch.tensor([prompt], dtype=torch.int32, device=dev)
    back = torch.empty((prompt, ROW), dtype=torch.bfloat16, device=dev)
    k3g.call("k3g_latent_mx8_gather", cache, prefix_table, 0, MX8_PAGE, pages, plen, back, prompt, s())
    torch.cuda.synchronize()
    rows = bf16_bits(slab).reshape(-1, ROW)[:prompt]
    host = np.zeros(pages * MX8_PAGE, dtype=np.uint8)
    put_rows(host, 0, MX8_PAGE, np.arange(prompt), rows)
    assert np.array_equal(cache.cpu().numpy(), host)
    assert np.array_equal(back.cpu().double().numpy(), mx8_rows(host, 0, MX8_PAGE, np.arange(pp), prompt)[0])

    table = (pp + torch.arange(B * max_pages, dtype=torch.int32, device=dev)).view(B, max_pages).contiguous()
    base = torch.tensor([59, 0, 61, 30], dtype=torch.int64, device=dev)                    # own tokens before the step
    for b in range(B):                                                                     # their latents
        old = normal_bf16(g, (int(base[b]), ROW))
        at = table[b].long().repeat_interleave(64)[:len(old)] * 64 + torch.arange(len(old), device=dev) % 64
        if len(old):
            k3g.call("k3g_latent_mx8_store", to_dev_bf16(old, dev), ROW, at, cache, 0, MX8_PAGE, pages, len(old), s())
    new_rows = torch.empty((B * S, ROW), dtype=torch.bfloat16, device=dev)
    q = torch.empty((B, S, heads, ROW), dtype=torch.bfloat16, device=dev)
    head = torch.randn((heads * LATENT, V), generator=tg, device=dev) * 0.1
    drafts = torch.empty((B, S - 1), dtype=torch.int64, device=dev); dprobs = torch.empty((B, S - 1, V), device=dev); u = torch.empty((B, S), device=dev)
    lens = torch.empty(B, dtype=torch.int32, device=dev)
    out = torch.empty((B, S, heads, LATENT), dtype=torch.bfloat16, device=dev)
    probs = torch.empty((B, S, V), device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev); tokens = torch.empty((B, S), dtype=torch.int64, device=dev)
    ws = torch.empty(k3g.latent_attn_workspace(B, S, heads), dtype=torch.uint8, device=dev)

    def step():
        pos = base[:, None] + torch.arange(S, device=dev)
        at = table.long().gather(1, pos // 64) * 64 + pos % 64
        k3g.call("k3g_latent_mx8_store", new_rows, ROW, at.view(-1), cache, 0, MX8_PAGE, pages, B * S, s())
        lens.copy_(base + S)
        k3g.call("k3g_latent_attn", q, heads * ROW, cache, 1, 0, MX8_PAGE, pages, prefix_table, plen, pp, table, lens, max_pages, out, ws, ws.numel(), B, S, heads, 0.07, s())
        probs.copy_(torch.softmax(out.view(B, S, heads * LATENT).float() @ head, -1))
        k3g.call("k3g_verify_draft", probs, V, dprobs, V, drafts, u, accepted, tokens, B, S - 1, V, s())
        base.add_(accepted + 1)

    def feed():
        new_rows.copy_(torch.randn(new_rows.shape, generator=tg, device=dev))
        q.copy_(1.4 * torch.randn(q.shape, generator=tg, device=dev))
        dprobs.copy_(torch.softmax(torch.randn(dprobs.shape, generator=tg, device=dev), -1))
        drafts.copy_(dprobs.view(-1, V).argmax(-1).view(B, S - 1))
        u.copy_(torch.rand(u.shape, generator=tg, device=dev) * 0.3)

    start = base.clone()
    feed()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    base.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    total = 0
    for _ in range(steps):
        feed()
        before = base.clone()
        graph.replay()
        torch.cuda.synchronize()
        hc, ht = cache.cpu().numpy(), table.cpu().numpy()
        hq = q.cpu().double().numpy()
        want, spread, ds = attn_oracle(hq, lambda t, n: mx8_rows(hc, 0, MX8_PAGE, t, n), np.arange(pp), prompt, ht, lens.cpu().numpy(), 0.07)
        assert np.all(np.abs(out.cpu().double().numpy() - want) <= attn_tolerance(want, spread, ds))
        o_acc, o_tok = verify_oracle(probs.cpu().numpy(), dprobs.cpu().numpy(), drafts.cpu().numpy(), u.cpu().numpy())
        assert np.array_equal(accepted.cpu().numpy(), o_acc) and np.array_equal(tokens.cpu().numpy(), o_tok)
        assert torch.equal(base, before + accepted + 1)
        total += int(accepted.sum())
    assert int(base.max()) > 64


@pytest.mark.parametrize("captured", [False, True])
def test_launched_behind_one_another_each_reads_what_the_one_before_wrote(k3g, dev, captured):
    """A chain without a wait of the host's: the token that verification draws is the slot of the row stored next, the cache is read back, attended to,
    and 150 times so, every time another row over the same pages.  Each output is what the same calls give with a wait after each."""
    import torch
    g = rng(34)
    pages, n, heads = 3, 150, 8
    V = pages * 64
    rows = to_dev_bf16(normal_bf16(g, (n, ROW)), dev)
    u = torch.rand((n, 1), device=dev, generator=torch.Generator(device=dev).manual_seed(34))
    target = torch.full((1, 1, V), 1.0 / V, device=dev)
    q = to_dev_bf16(normal_bf16(g, (1, 1, heads, ROW)), dev)
    table, lens = torch.tensor([2, 0, 1], dtype=torch.int32, device=dev), torch.tensor([V], dtype=torch.int32, device=dev)
    start = torch.zeros(pages * MX8_PAGE, dtype=torch.uint8, device=dev)
    k3g.call("k3g_latent_mx8_store", to_dev_bf16(normal_bf16(g, (V, ROW)), dev), ROW, torch.arange(V, device=dev), start, 0, MX8_PAGE, pages, V, k3g.current_stream())
    cache = torch.empty_like(start)
    accepted, token = torch.empty(1, dtype=torch.int32, device=dev), torch.empty((1, 1), dtype=torch.int64, device=dev)
    ws = torch.empty(k3g.latent_attn_workspace(1, 1, heads), dtype=torch.uint8, device=dev)

    def chain(tokens, back, out, stop):
        cache.copy_(start)
        for i in range(n):
            s = k3g.current_stream()
            k3g.call("k3g_verify_draft", target, V, None, V, token, u[i], accepted, token, 1, 0, V, s)
            stop()
            k3g.call("k3g_latent_mx8_store", rows[i], ROW, token, cache, 0, MX8_PAGE, pages, 1, s)
            stop()
            k3g.call("k3g_latent_mx8_gather", cache, table, 0, MX8_PAGE, pages, lens, back[i], V, s)
            stop()
            k3g.call("k3g_latent_attn", q, heads * ROW, cache, 1, 0, MX8_PAGE, pages, None, None, 0, table, lens, pages, out[i], ws, ws.numel(), 1, 1, heads, 0.07, s)
            stop()
            tokens[i].copy_(token.view(-1))

    def outputs():
        return (torch.zeros((n, 1), dtype=torch.int64, device=dev), torch.zeros((n, V, ROW), dtype=torch.bfloat16, device=dev),
                torch.zeros((n, heads, LATENT), dtype=torch.bfloat16, device=dev))
    want, got = outputs(), outputs()
    chain(*want, torch.cuda.synchronize)
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            chain(*got, lambda: None)
        graph.replay()
    else:
        chain(*got, lambda: None)
    torch.cuda.synchronize()
    assert len(torch.unique(want[0])) > 50
    for a, b in zip(want, got):
        assert torch.equal(a.view(torch.int64 if a.dtype == torch.int64 else torch.int16), b.view(torch.int64 if b.dtype == torch.int64 else torch.int16))
