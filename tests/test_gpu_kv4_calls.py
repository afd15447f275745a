"""GPU: calls over a 4-bit cache that combine what the other tests take one by one: per-token score modifications, draft trees within a
window, block-table offsets, appends to given rows of q, pages of three tiles, and a captured step with positions of several axes."""

import ctypes

import numpy as np
import pytest

import kv4_format as f4
from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.kv4 import KV4Pool
from exactattention_amd.serving import DecodeGraph, ExactAttentionBackend, HeadNorm, PagedKVCache, Rotary
from gen import bf16
from test_gpu_kv4 import _problem
from test_gpu_kv4_run import _Loop, _bits

pytestmark = pytest.mark.gpu


def _same_bits(pair, mods, out="bf16"):
    """The step over the 4-bit cache against the bf16 kernels on its values."""
    ab = default_alpha_bits(pair[1]["geom"]["head_dim"])
    want, wf, _ = hip.attention_problem(pair[1], None, out, alpha_bits=ab, kernel="general", mods=mods, device="cuda:0")
    got, flags, _ = hip.attention_problem(pair[0], None, out, alpha_bits=ab, mods=mods, device="cuda:0")
    assert not flags.any() and not wf.any() and np.array_equal(got, want)


@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("B,T,Hkv,grp,d", [(3, 1, 2, 2, 128), (2, 5, 2, 2, 72), (16, 64, 4, 2, 128)])
@pytest.mark.parametrize("what", ["documents", "documents, bias", "bias elsewhere, cap"])
def test_modifications_by_token(gpu, what, B, T, Hkv, grp, d, out):
    """First keys and positions of each token: documents packed into a sequence, and distances from other places than the prefix's
    end. Rows whose document starts past their prefix see nothing."""
    rng = np.random.default_rng(B + T + d)
    S = T + 150
    pair = _problem(rng, B, T, Hkv * grp, Hkv, S, d, 32, qscale=2.0)
    kv = np.broadcast_to(S - T + 1 + np.arange(T), (B, T))
    begin = np.minimum((kv // 47) * 47, kv - 1).astype(np.int32)
    begin[0, 0] = kv[0, 0]  # nothing
    slopes = (1.4426950408889634 * 2.0 ** (-2.0 * (np.arange(Hkv * grp) % 4 + 1))).astype(np.float32)
    pos = rng.integers(0, S, (B, T)).astype(np.int32)
    mods = {"documents": dict(kv_begin=begin), "documents, bias": dict(kv_begin=begin, slopes=slopes),
            "bias elsewhere, cap": dict(slopes=slopes, q_pos=pos, softcap=25.0)}[what]
    _same_bits(pair, hip.ScoreMods(**mods), out)


@pytest.mark.parametrize("B,T,Hkv,grp", [(2, 16, 2, 2), (8, 64, 8, 2)])
@pytest.mark.parametrize("begin", [False, True])
def test_trees(gpu, B, T, Hkv, grp, begin):
    """Draft trees over long prefixes, alone and behind a first key, in blocks of 4 and of 16 rows; the prefix ends inside a tile."""
    rng = np.random.default_rng(T + grp)
    L = 203
    mask = np.zeros((B, T), np.uint64)
    for b in range(B):
        parents = [-1] + [int(rng.integers(-1, i)) for i in range(1, T)]
        for i in range(T):
            j = i
            while j >= 0:
                mask[b, i] |= np.uint64(1 << j)
                j = parents[j]
    pair = _problem(rng, B, T, Hkv * grp, Hkv, L + T, 128, 64, kv_len=np.full((B, T), L), tree=(mask, np.full(B, L, np.int32)))
    if begin:
        _same_bits(pair, hip.ScoreMods(kv_begin=rng.integers(150, L + 1, (B, T)).astype(np.int32)))
    else:
        _same_bits(pair, None)


def test_block_table_offsets(gpu):
    """Sequences that find their part of the block table by an offset, in another order than the batch's."""
    rng = np.random.default_rng(2)
    B, T, S = 4, 3, 130
    pair = _problem(rng, B, T, 4, 2, S, 96)
    per = pair[1]["block_table"].shape[1]
    order = np.array([2, 0, 3, 1])
    moved = tuple({**p, "block_table": p["block_table"][order], "block_table_offset": np.argsort(order).astype(np.int64) * per}
                  for p in pair)
    ab = default_alpha_bits(96)
    want = hip.attention_problem(pair[1], None, alpha_bits=ab, device="cuda:0")[0]
    for p in moved:
        got, flags, _ = hip.attention_problem(p, None, alpha_bits=ab, device="cuda:0")
        assert not flags.any() and np.array_equal(got, want)


def test_append_to_rows_of_q(gpu):
    """q to given rows of a larger tensor, positions from an offset, tokens without a slot or a row of q."""
    import torch
    g = torch.Generator().manual_seed(1)
    n, hq, hk, d = 40, 6, 2, 96
    q, k, v = (torch.randn((n, h, d), generator=g).bfloat16().cuda() for h in (hq, hk, hk))
    rot = Rotary(d, rot_dim=48, device="cuda:0")
    norm = HeadNorm(*((1 + 0.2 * torch.randn(d, generator=g)).cuda() for _ in range(2)))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    dst = torch.randperm(64, generator=g)[:n].cuda()
    dst[5] = -1
    rows = torch.randperm(100, generator=g)[:n].cuda()
    rows[7], rows[8] = -1, 100
    a, b = KV4Pool(4, 16, hk, d, "cuda:0"), KV4Pool(4, 16, hk, d, "cuda:0")
    out = torch.full((100, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    got = rot.append(q, k, v, pos, dst, a, q_rows=rows, q_out=out, pos_offset=9, norm=norm)
    want = rot.append(q, k, v, pos + 9, dst, b, norm=norm)
    assert got.data_ptr() == out.data_ptr()
    live = (rows >= 0) & (rows < 100)
    assert torch.equal(out[rows[live]], want[live])
    rest = torch.ones(100, dtype=torch.bool, device="cuda")
    rest[rows[live]] = False
    assert bool((out[rest] == 7.0).all())
    for x, y in zip((a.k, a.k_scales, a.v, a.v_scales), (b.k, b.k_scales, b.v, b.v_scales)):
        assert torch.equal(x, y)


def test_pages_of_three_tiles(gpu):
    """The C entry point on pages of 48 slots, which are no power of two: rows to the bit, the others left alone."""
    import torch
    rng = np.random.default_rng(3)
    n, H, d, P, pages = 100, 2, 72, 48, 3
    w = f4.width(d)
    x = [torch.from_numpy(rng.standard_normal((n, H, d)).astype(np.float32)).cuda() for _ in range(2)]
    dst = rng.permutation(pages * P)[:n].astype(np.int64)
    k, ks = (torch.full((pages, H, P, m), 0x5A, dtype=torch.uint8, device="cuda") for m in (w // 2, w // 32))
    v, vs = (torch.full((pages, H, P // 16, m, 16), 0x5A, dtype=torch.uint8, device="cuda") for m in (w // 2, w // 32))
    to = torch.from_numpy(dst).cuda()
    r = hip.RotaryArgs(num_tokens=n, num_kv_heads=H, head_dim=d, num_axes=1, in_fp32=1, scale=1.0, k_tok_stride=H * d, k_head_stride=d,
                       v_tok_stride=H * d, v_head_stride=d, ko_tok_stride=w, ko_head_stride=P * w, vo_tok_stride=w, vo_head_stride=P * w,
                       pool_rows=pages * P, k=x[0].data_ptr(), v=x[1].data_ptr(), dst_rows=to.data_ptr(), k_out=k.data_ptr(),
                       v_out=v.data_ptr())
    a = hip.NormRotaryArgs(r=r, k_scales=ks.data_ptr(), v_scales=vs.data_ptr(), k_page_stride=H * P * w, v_page_stride=H * P * w, page_size=P)
    lib = hip.load()
    assert lib.ea_hip_norm_rotary(ctypes.byref(a), hip._stream_ptr(torch)) == 0
    torch.cuda.synchronize()
    rows = [k, ks, *(t.transpose(3, 4).flatten(2, 3) for t in (v, vs))]
    page, slot = dst // P, dst % P
    for src, codes, scales in ((x[0], *rows[:2]), (x[1], *rows[2:])):
        c, s = f4.quantize(src.double().cpu().numpy())
        codes, scales = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
        assert np.array_equal(scales[page, :, slot], s)
        assert np.array_equal(codes[page, :, slot][..., :d // 2], c[..., :d // 2])
        codes[page, :, slot] = 0x5A
        scales[page, :, slot] = 0x5A
        assert np.all(codes == 0x5A) and np.all(scales == 0x5A)


@pytest.mark.parametrize("window", [0, 30])
def test_verify_tree_within_a_window(gpu, window):
    """The backend's draft tree over a 4-bit cache, with norms and rotary positions: a window counts the path's nodes and the
    prefix's last keys."""
    import torch
    L = _Loop(mods=dict(window=window) if window else dict(softcap=30.0), d=64)
    c, s, N = L.c, L.seqs[0], 10
    L.be.prefill(s, *L.new(75))
    n0 = c.length[s]
    parents = [-1, 0, 1, 2, -1, 4, 3, 6, 7, 8]
    depth = []
    for p in parents:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    q, k, v = L.new(N)
    out, flags = L.be.verify_tree(s, q, k, v, parents)
    assert not flags.any()
    mask = np.zeros((1, N), np.uint64)
    for i in range(N):
        j = i
        while j >= 0 and not (window and depth[i] - depth[j] >= window):
            mask[0, i] |= np.uint64(1 << j)
            j = parents[j]
    kk, vv = ((x.view(torch.int16).cpu().numpy().view(np.uint16)[c.pages[s]].transpose(1, 0, 2, 3).reshape(L.Hkv, -1, L.d)
               [:, :c.length[s]]) for x in c.pool4.values())
    p = problem.contiguous(L.q_of(q, n0 + np.array(depth))[None], kk[None], vv[None], np.full((1, N), n0), tree_mask=mask, tree_base=[n0])
    begin = np.clip(n0 + np.array(depth) + 1 - window, 0, n0).astype(np.int32)[None]
    m = hip.ScoreMods(kv_begin=begin) if window else hip.ScoreMods(softcap=30.0)
    want = hip.attention_problem(p, None, alpha_bits=default_alpha_bits(64), mods=m, device="cuda:0")[0][0]
    assert np.array_equal(out, want)


def test_captured_step_with_positions_of_several_axes(gpu):
    """A captured decode step over a 4-bit cache with norms and three position axes, replayed between eager work."""
    import torch
    d, Hq, Hkv, B = 128, 8, 2, 3
    g = torch.Generator().manual_seed(5)
    rot = Rotary(d, sections=[24, 20, 20], device="cuda:0")
    norm = HeadNorm(*((1 + 0.2 * torch.randn(d, generator=g)).bfloat16().cuda() for _ in range(2)))
    bes, seqs = [], []
    for _ in range(2):
        c = PagedKVCache(60, 16, Hkv, d, B, 200, bits=4)
        bes.append(ExactAttentionBackend(c, Hq, alpha_bits=default_alpha_bits(d), rotary=rot, norm=norm))
        seqs.append([c.add_sequence() for _ in range(B)])
    ql = [40, 5, 17]
    new = lambda n: [torch.randn((n, h, d), generator=g).bfloat16().cuda() for h in (Hq, Hkv, Hkv)]  # noqa: E731
    first, pos = new(sum(ql)), torch.randint(0, 500, (3, sum(ql)), generator=g, dtype=torch.int32).cuda()
    for be, s in zip(bes, seqs):
        be.check_flags(be.forward(*first, s, ql, positions=pos)[1])
    torch.cuda.synchronize()
    graph = DecodeGraph(bes[0], seqs[0], max_len=150)
    for i in range(5):
        q, k, v = new(B)
        pos = torch.randint(0, 500, (3, B), generator=g, dtype=torch.int32).cuda()
        for t, x in ((graph.q, q[:, None]), (graph.k, k), (graph.v, v)):
            t.copy_(x.view(torch.int16))
        graph.positions.copy_(pos)
        out, flags = graph.step()
        graph.check_flags(flags)
        want, wf = bes[1].forward(q, k, v, seqs[1], [1] * B, positions=pos)
        bes[1].check_flags(wf)
        assert np.array_equal(_bits(out), _bits(want)), i
    graph.close()


def test_pool_takes_strided_keys(gpu):
    """Keys and values as parts of one projection, with strides over tokens and heads, int16 or bf16; a single head of any stride."""
    import torch
    rng = np.random.default_rng(9)
    n, H, d = 50, 3, 64
    fused = torch.from_numpy(bf16(rng, (n, 2 * H * d + 40)).view(np.int16)).cuda()
    k, v = fused[:, 8:8 + H * d].view(n, H, d), fused[:, 40 + H * d:].view(n, H, d)
    dst = torch.arange(n, device="cuda")
    a, b = KV4Pool(4, 16, H, d, "cuda:0"), KV4Pool(4, 16, H, d, "cuda:0")
    a.append(k, v, dst)
    b.append(k.contiguous().view(torch.bfloat16), v.contiguous().view(torch.bfloat16), dst)
    for x, y in zip((a.k, a.k_scales, a.v, a.v_scales), (b.k, b.k_scales, b.v, b.v_scales)):
        assert torch.equal(x, y)
    off = fused[:, 1:1 + H * d].view(n, H, d)  # rows that start on 2 bytes
    a.append(off, off, dst)
    b.append(off.contiguous(), off.contiguous(), dst)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.k_scales, b.k_scales)
