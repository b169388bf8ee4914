"""Refusals of the latent-cache and draft-verification entries, answered before any CUDA call, and their oracles checked on
cases small enough to do by hand.  No GPU."""
import numpy as np
import pytest

import k3o
from latent_util import LATENT, MX8_PAGE, PAGE, ROW, attn_oracle, mx8_rows, put_rows, verify_oracle
from util import normal_bf16, rng

P = 4096                                                        # an aligned address that nothing dereferences


def _with(base, **change):
    args = dict(base)
    args.update(change)
    return list(args.values())


STORE = dict(rows=P, row_stride=576, slots=P, cache=P, layer_off=0, page_stride=MX8_PAGE, pages=4, T=1, stream=None)
GATHER = dict(cache=P, table=P, layer_off=0, page_stride=MX8_PAGE, pages=4, lens=P, out=P, n=1, stream=None)
ATTN = dict(q=P, q_stride=24 * ROW, cache=P, mx8=1, layer_off=0, page_stride=MX8_PAGE, pages=4, prefix_table=P, prefix_len=P, prefix_pages=1,
            table=P, lens=P, max_pages=1, out=P, workspace=P, bytes=1 << 40, B=1, S=1, heads=24, scale=0.1, stream=None)
VERIFY = dict(target=P, target_stride=100, draft=P, draft_stride=100, ids=P, u=P, accepted=P, tokens=P, B=1, S=2, V=100, stream=None)


@pytest.mark.parametrize("name,base,change,code", [
    ("k3g_latent_mx8_store", STORE, dict(rows=None), -1), ("k3g_latent_mx8_store", STORE, dict(slots=None), -1),
    ("k3g_latent_mx8_store", STORE, dict(rows=P + 8), -3), ("k3g_latent_mx8_store", STORE, dict(row_stride=580), -3),
    ("k3g_latent_mx8_store", STORE, dict(row_stride=568), -2), ("k3g_latent_mx8_store", STORE, dict(layer_off=16), -3), ("k3g_latent_mx8_store", STORE, dict(cache=P + 16), -3),
    ("k3g_latent_mx8_store", STORE, dict(page_stride=MX8_PAGE + 8), -3), ("k3g_latent_mx8_store", STORE, dict(page_stride=MX8_PAGE - 32), -2),
    ("k3g_latent_mx8_store", STORE, dict(layer_off=32), -2), ("k3g_latent_mx8_store", STORE, dict(layer_off=-32), -2),
    ("k3g_latent_mx8_store", STORE, dict(T=-1), -2), ("k3g_latent_mx8_store", STORE, dict(pages=-1), -2), ("k3g_latent_mx8_store", STORE, dict(T=0), 0),
    ("k3g_latent_mx8_gather", GATHER, dict(lens=None), -1), ("k3g_latent_mx8_gather", GATHER, dict(out=P + 4), -3),
    ("k3g_latent_mx8_gather", GATHER, dict(page_stride=32), -2), ("k3g_latent_mx8_gather", GATHER, dict(cache=P + 16), -3), ("k3g_latent_mx8_gather", GATHER, dict(n=-1), -2), ("k3g_latent_mx8_gather", GATHER, dict(n=0), 0),
    ("k3g_latent_attn", ATTN, dict(q=None), -1), ("k3g_latent_attn", ATTN, dict(lens=None), -1), ("k3g_latent_attn", ATTN, dict(prefix_table=None), -1),
    ("k3g_latent_attn", ATTN, dict(prefix_len=None), -1), ("k3g_latent_attn", ATTN, dict(table=None), -1), ("k3g_latent_attn", ATTN, dict(workspace=None), -1),
    ("k3g_latent_attn", ATTN, dict(q=P + 2), -3), ("k3g_latent_attn", ATTN, dict(cache=P + 16), -3), ("k3g_latent_attn", ATTN, dict(q_stride=24 * ROW + 4), -3), ("k3g_latent_attn", ATTN, dict(workspace=P + 8), -3),
    ("k3g_latent_attn", ATTN, dict(mx8=0, page_stride=PAGE * ROW + 4), -3), ("k3g_latent_attn", ATTN, dict(mx8=0, page_stride=PAGE * ROW - 16), -2), ("k3g_latent_attn", ATTN, dict(mx8=0, layer_off=8, page_stride=2 * PAGE * ROW), -3),
    ("k3g_latent_attn", ATTN, dict(q_stride=23 * ROW), -2), ("k3g_latent_attn", ATTN, dict(S=0), -2), ("k3g_latent_attn", ATTN, dict(heads=0), -2),
    ("k3g_latent_attn", ATTN, dict(B=-1), -2), ("k3g_latent_attn", ATTN, dict(max_pages=-1), -2), ("k3g_latent_attn", ATTN, dict(B=4097), -5),
    ("k3g_latent_attn", ATTN, dict(S=32769, heads=1, q_stride=ROW), -5), ("k3g_latent_attn", ATTN, dict(max_pages=(1 << 20) + 1), -5),
    ("k3g_latent_attn", ATTN, dict(prefix_pages=(1 << 20) + 1), -5), ("k3g_latent_attn", ATTN, dict(prefix_pages=-1), -2), ("k3g_latent_attn", ATTN, dict(pages=1 << 31), -2),
    ("k3g_latent_attn", ATTN, dict(scale=float("nan")), -4), ("k3g_latent_attn", ATTN, dict(scale=float("-inf")), -4), ("k3g_latent_attn", ATTN, dict(scale=3e38, bytes=0), -6),
    ("k3g_latent_attn", ATTN, dict(bytes=0), -6), ("k3g_latent_attn", ATTN, dict(B=0), 0),
    ("k3g_verify_draft", VERIFY, dict(target=None), -1), ("k3g_verify_draft", VERIFY, dict(ids=None), -1), ("k3g_verify_draft", VERIFY, dict(target=P + 4), -3),
    ("k3g_verify_draft", VERIFY, dict(draft=P + 4), -3), ("k3g_verify_draft", VERIFY, dict(target_stride=99), -2), ("k3g_verify_draft", VERIFY, dict(draft_stride=99), -2),
    ("k3g_verify_draft", VERIFY, dict(V=0), -2), ("k3g_verify_draft", VERIFY, dict(S=-1), -2), ("k3g_verify_draft", VERIFY, dict(S=33), -5), ("k3g_verify_draft", VERIFY, dict(B=0), 0)])
def test_refusals(k3g, name, base, change, code):
    assert k3g.raw(name, *_with(base, **change)) == code


def test_workspace_query(k3g):
    sizes = [k3g.latent_attn_workspace(b, s, h) for b, s, h in ((1, 1, 1), (8, 1, 24), (8, 4, 24), (64, 4, 96))]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for shape in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (4097, 1, 1), (1, 32769, 1)):
        with pytest.raises(k3g.K3gError):
            k3g.latent_attn_workspace(*shape)
    with pytest.raises(k3g.K3gError, match="EWORKSPACE"):
        k3g.call("k3g_latent_attn", *_with(ATTN, bytes=k3g.latent_attn_workspace(1, 1, 24) - 1))


def test_mx8_oracle_round_trip():
    """A row put into the oracle's cache and read back: half an E4M3 step of its block's scale away at most, bf16 exactly in the rope columns."""
    g = rng(5)
    rows = normal_bf16(g, (70, ROW))
    cache = np.zeros(3 * 2 * MX8_PAGE, dtype=np.uint8)
    slots = np.concatenate([g.permutation(128)[:70] + 64])
    put_rows(cache, MX8_PAGE, 2 * MX8_PAGE, slots, rows)
    assert not cache[:2 * MX8_PAGE].any()                        # page 0 holds none of the slots
    back, held = mx8_rows(cache, MX8_PAGE, 2 * MX8_PAGE, np.array([0, 1, 2]), 192)
    x, y = k3o.bf16_to_f32(rows).astype(np.float64), back[slots]
    assert held.all() and np.array_equal(x[:, LATENT:], y[:, LATENT:])
    # normal codes: 2^-4 relative; below 2^-6 * scale the step is fixed, half of it 2^-10 * scale <= 2^-10 * amax / 224
    amax = np.abs(x[:, :LATENT]).reshape(-1, 16, 32).max(-1).repeat(32, -1).reshape(-1, LATENT)
    assert np.all(np.abs(x[:, :LATENT] - y[:, :LATENT]) <= 2.0 ** -4 * np.abs(x[:, :LATENT]) + 2.0 ** -10 * amax / 224)


def test_attn_oracle_on_one_visible_token():
    g = rng(6)
    q, k = g.standard_normal((2, 2, 3, ROW)), g.standard_normal((64, ROW))
    out, spread, _ = attn_oracle(q, lambda t, n: (k[:n], np.ones(n, dtype=bool)), None, 0, np.zeros((2, 1), dtype=np.int32), [2, 0], 0.1)
    assert np.allclose(out[0, 0], k[0, :LATENT]) and np.allclose(spread[0, 0], np.abs(k[0, :LATENT]))   # step 0 of 2 sees token 0 alone
    assert not out[1].any()                                                                             # nothing to see


def test_verify_oracle_gives_back_the_target_distribution():
    """Over a grid of random numbers the first token's distribution is the target's, whatever the draft model's was."""
    V, n = 4, 24
    p, q = np.array([0.5, 0.25, 0.125, 0.125], dtype=np.float32), np.array([0.125, 0.25, 0.5, 0.125], dtype=np.float32)
    u = (np.arange(n) + 0.5) / n
    count = np.zeros(V)
    for x in range(V):
        a, r = np.meshgrid(u, u)
        grid = np.stack([a.ravel(), r.ravel()], 1).astype(np.float32)
        B = len(grid)
        _, tok = verify_oracle(np.broadcast_to(p, (B, 2, V)), np.broadcast_to(q, (B, 1, V)), np.full((B, 1), x), grid)
        count += q[x] * np.bincount(tok[:, 0], minlength=V) / B
    assert np.allclose(count, p, atol=1e-9)                      # the grid's 24 points divide every boundary evenly


def test_warps_shares_of_registers_are_what_the_attention_is_launched_with(tmp_path):
    """The warps of the attention kernel divide the registers that its block is launched with; a compiler that gave it fewer would leave
    setmaxnreg.inc waiting for good.  The shares are read from the source, the launch from what ptxas prints."""
    import os
    import re
    import shutil
    import subprocess
    import sys
    nvcc = os.environ.get("NVCC", "nvcc")
    if not shutil.which(nvcc):
        pytest.skip("no nvcc")
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kern-k3_b200")
    sys.path.insert(0, here)
    import build
    source = open(os.path.join(here, "csrc", "latent_attn.cu")).read()
    softmax, loaders = (int(x) for x in re.findall(r"setmaxnreg\.inc\.sync\.aligned\.u32 (\d+)", source))
    rest, = (int(x) for x in re.findall(r"setmaxnreg\.dec\.sync\.aligned\.u32 (\d+)", source))
    sizes = {k: int(v) for k, v in re.findall(r"(kSoftmax|kLoaders) = (\d+)", source)}
    r = subprocess.run([nvcc] + build.ARCH + build.COMMON + ["-Xptxas", "-v", "-cubin", "-I", os.path.join(here, "..", "include"), os.path.join(here, "csrc", "latent_attn.cu"),
                                                             "-o", str(tmp_path / "attn.cubin")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    used = [int(n) for n in re.findall(r"Compiling entry function '\S*latent_attn_kernel\S*'.*?Used (\d+) registers", r.stdout + r.stderr, re.S)]
    assert len(used) == 2
    threads = sizes["kSoftmax"] + sizes["kLoaders"] + 128
    for n in used:
        assert sizes["kSoftmax"] * softmax + sizes["kLoaders"] * loaders + 128 * rest <= threads * ((n + 7) // 8 * 8)


@pytest.mark.parametrize("name", ["latent_attn.cu", "latent_cache.cu", "latent_page.cuh", "verify.cu"])
def test_kernels_launched_behind_others_load_coherently(name):
    """They begin while the launch before them still writes: nothing that they read is read-only for as long as they run, so no load of theirs may take
    the path that asks for it (nor be given it by the compiler, for const __restrict__)."""
    import os
    import re
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source = open(os.path.join(here, "kern-k3_b200", "csrc", name)).read()
    source = re.sub(r"//[^\n]*", "", source)
    assert not re.findall(r"__ldg\b|ld\.global\.nc|ld_stream(?:32|_vec<\d+>)?\(|ld_keep\w*|__restrict__", source)
