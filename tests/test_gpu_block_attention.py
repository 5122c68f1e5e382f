"""block_attention's operators on an MI355X against their definition in 64 bits (oracle/block_attn_ref.py): integers equal, the append bit for bit what
apply_rope_pos_ids and set_kv_cache write, attention within the output's half step and the bound that the oracle derives for fp32 work."""
import numpy as np
import pytest
import torch

from oracle import block_attn_ref as R

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from vox_serve_amd import _native as N
    N.ctx()
    return torch.device("cuda", torch.cuda.current_device())


def f64(t):
    return t.detach().cpu().double().numpy()


class Paged:
    """Requests of the given lengths on shuffled pages, new rows at their ends, a page that is nobody's."""

    def __init__(self, dev, dtype, h, d, page, kv_lens, q_lens, seed=0, spare=1):
        g = torch.Generator().manual_seed(seed)
        self.kv_lens, self.page = kv_lens, page
        need = [-(-n // page) for n in kv_lens]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.pages, at = [], 0
        for n in need:
            self.pages.append(order[at:at + n])
            at += n
        self.indptr = torch.tensor([0] + list(np.cumsum(need)), dtype=torch.int32, device=dev)
        self.indices = torch.tensor(order[:max(at, 1)], dtype=torch.int32, device=dev)
        self.req = [r for r, m in enumerate(q_lens) for _ in range(m)]
        self.kvlen = [kv_lens[r] - m + i + 1 for r, m in enumerate(q_lens) for i in range(m)]
        self.n = len(self.req)
        self.q_req = torch.tensor(self.req, dtype=torch.int32, device=dev)
        self.q_kvlen = torch.tensor(self.kvlen, dtype=torch.int32, device=dev)
        self.row_page = torch.tensor([self.pages[r][(n - 1) // page] for r, n in zip(self.req, self.kvlen)], dtype=torch.int32, device=dev)
        self.row_slot = torch.tensor([(n - 1) % page for n in self.kvlen], dtype=torch.int32, device=dev)
        self.kv = torch.randn(total, 2, page, h, d, generator=g).to(dtype).to(dev)
        self.gen, self.dtype, self.dev, self.h, self.d = g, dtype, dev, h, d

    def rnd(self, *shape, s=1.0):
        return (s * torch.randn(*shape, generator=self.gen)).to(self.dtype).to(self.dev)

    @property
    def plan(self):
        return self.q_req, self.q_kvlen, self.indptr, self.indices

    def bounds(self, block):
        """Of every complete block, by the oracle."""
        k = f64(self.kv)[:, 0]
        total, page, h, d = k.shape
        per = page // block
        b, s = np.zeros((total, h, per, 2, d), np.int8), np.zeros((total, h, per), np.float32)
        for p in range(total):
            for g in range(h):
                for j in range(per):
                    b[p, g, j], s[p, g, j] = R.bounds(k[p, j * block:(j + 1) * block, g])
        return torch.from_numpy(b).to(self.dev), torch.from_numpy(s).to(self.dev)


def table(dev, length, half, theta=1e4):
    a = torch.arange(length, dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    return torch.stack([a.cos(), a.sin()], -1).float().to(dev)


# ---------------------------------------------------------------- append
APPEND = [  # heads, kv heads, dim, page, block, rot, pairs interleaved, kv lengths, new rows
    (16, 8, 128, 128, 64, 128, False, [200, 64, 128, 1], [1, 1, 1, 1]),
    (32, 2, 128, 64, 64, 64, True, [64, 63, 65], [1, 1, 1]),
    (14, 2, 64, 48, 16, 64, False, [48, 100, 17, 3], [48, 37, 17, 1]),
    (8, 8, 64, 16, 16, 32, True, [33, 16], [33, 1]),
    (12, 4, 128, 32, 32, 0, False, [70, 32], [70, 32]),
    (4, 1, 128, 128, 128, 128, True, [300], [300]),
    (4, 2, 64, 32, 16, 18, False, [40], [40]),           # an odd number of pairs: no vector of eight fits
    (4, 2, 64, 32, 16, 6, True, [40, 2], [40, 2]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,h,d,page,block,rot,interleave,kv_lens,q_lens", APPEND)
def test_rope_append(dev, dtype, hq, h, d, page, block, rot, interleave, kv_lens, q_lens):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, TYPES[dtype], h, d, page, kv_lens, q_lens, seed=hq + rot)
    qkv = s.rnd(s.n, (hq + 2 * h) * d)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, h * d, h * d], 1))
    pos = torch.tensor([n - 1 for n in s.kvlen], dtype=torch.int32, device=dev)
    cs = table(dev, 64, rot // 2) if rot else None        # shorter than some positions: those take the last row
    before = s.kv.clone()
    for n_req in (0, len(q_lens)):
        s.kv.copy_(before)
        bounds, steps = B.new_bounds(s.kv, block)
        got = B.rope_append(q, k, v, s.kv, cs, pos, s.row_page, s.row_slot, interleave=interleave, bounds=bounds, steps=steps, n_req=n_req)
        tab = cs.cpu().numpy() if rot else np.zeros((1, 0, 2), np.float32)
        half_step = torch.finfo(TYPES[dtype]).eps / 2
        tiny = torch.finfo(TYPES[dtype]).smallest_normal * half_step
        for x, y in ((q, got), (k, None)):
            want = R.rotate(f64(x), tab, pos.cpu().numpy(), interleave)
            have = f64(got) if y is not None else f64(s.kv[s.row_page.long(), 0, s.row_slot.long()])
            # two products in fp32, each off by 2^-24 of |x| + |y| <= 2 max|x| at most, then one rounding
            far = np.abs(have - want)
            assert (far <= half_step * np.abs(want) * (1 + half_step) + 2.0 ** -22 * np.abs(f64(x)).max(-1, keepdims=True) + tiny).all()
        assert torch.equal(s.kv[s.row_page.long(), 1, s.row_slot.long()], v)
        # nothing else of the cache has changed
        mask = torch.zeros(s.kv.shape[0], page, dtype=torch.bool, device=dev)
        mask[s.row_page.long(), s.row_slot.long()] = True
        assert torch.equal(s.kv.transpose(1, 2)[~mask], before.transpose(1, 2)[~mask])
        # bounds: of the blocks that were completed, of no others
        want_b, want_s = s.bounds(block)
        done = torch.zeros(s.kv.shape[0], page // block, dtype=torch.bool, device=dev)
        last = (s.row_slot.long() + 1) % block == 0
        done[s.row_page.long()[last], s.row_slot.long()[last] // block] = True
        assert torch.equal(bounds.transpose(1, 2)[done], want_b.transpose(1, 2)[done]) and torch.equal(steps.transpose(1, 2)[done], want_s.transpose(1, 2)[done])
        assert not bounds.transpose(1, 2)[~done].any() and not steps.transpose(1, 2)[~done].any()


@pytest.mark.parametrize("hq,h,d,rot,interleave,n", [(16, 8, 128, 128, False, 3), (32, 2, 128, 64, True, 70), (14, 2, 64, 64, False, 150), (4, 2, 16, 8, True, 5), (4, 2, 24, 22, False, 9),
                                                     (16, 8, 128, 64, False, 33)])
def test_rope_append_is_rope_then_append(dev, hq, h, d, rot, interleave, n):
    from vox_serve_amd import block_attention as B
    from vox_serve_amd.flashinfer_utils import FlashInferPrefillWrapper, _rope_table, apply_rope_pos_ids
    page = 32
    need = -(-n // page)
    g = torch.Generator().manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)
    q, k, v = r(n, hq, d), r(n, h, d), r(n, h, d)
    w = FlashInferPrefillWrapper(None, hq, h, hq * d, page, device=dev)
    w.plan(torch.tensor([0, n]), torch.tensor([0, need]), torch.randperm(need, generator=g).int(), torch.tensor([n - (need - 1) * page]), torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int32, device=dev) * 37
    qr, kr = apply_rope_pos_ids(q, k, pos, interleave=interleave, rope_theta=1e6, rotary_dim=rot)
    want, have = torch.zeros(need, 2, page, h, d, dtype=torch.bfloat16, device=dev), torch.zeros(need, 2, page, h, d, dtype=torch.bfloat16, device=dev)
    w.set_kv_cache(want, kr, v)
    cs = _rope_table(dev, 8192, rot, 1e6, 1.0, None).view(8192, rot // 2, 2)
    assert torch.equal(w.set_kv_cache_rope(have, q, k, v, pos, cs, interleave=interleave), qr)
    assert torch.equal(have, want)
    # q turned where it is
    have.zero_()
    q2 = q.clone()
    assert B.rope_append(q2, k, v, have, cs, pos.long(), w.token_to_page, w.token_to_cache, interleave=interleave, out=q2) is q2
    assert torch.equal(q2, qr) and torch.equal(have, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,rot,interleave", [(128, 128, False), (64, 64, True), (128, 64, False)])
def test_rope_append_rounds_where_it_says(dev, dtype, d, rot, interleave):
    """x cos rounded to 32 bits, the fused sum rounded to 32, then to the type: the bits of that, over enough values that another order would show."""
    from vox_serve_amd import block_attention as B
    n, hq, h, page = 600, 16, 8, 64
    s = Paged(dev, TYPES[dtype], h, d, page, [n], [n], seed=d)
    q, k = s.rnd(n, hq, d), s.rnd(n, h, d)
    cs = table(dev, n, rot // 2)
    got = B.rope_append(q, k, k, s.kv, cs, s.q_kvlen - 1, s.row_page, s.row_slot, interleave=interleave)
    c, sn = (cs[:, None, :, i].cpu().numpy() for i in (0, 1))
    for x, y in ((q, got), (k, s.kv[s.row_page.long(), 0, s.row_slot.long()])):
        f = x.float().cpu().numpy()
        a, b = (f[..., 0:rot:2], f[..., 1:rot:2]) if interleave else (f[..., :rot // 2], f[..., rot // 2:rot])
        u = ((a * c).astype(np.float64) - b.astype(np.float64) * sn).astype(np.float32)       # (products of 8 or 11 by 24 bits are exact in 64)
        v = ((b * c).astype(np.float64) + a.astype(np.float64) * sn).astype(np.float32)
        turned = np.stack([u, v], -1).reshape(n, x.shape[1], rot) if interleave else np.concatenate([u, v], -1)
        want = torch.cat([torch.from_numpy(turned).to(TYPES[dtype]), x[..., rot:].cpu()], -1)
        assert torch.equal(y.cpu(), want)


def test_rope_append_passes_rows_over(dev):
    from vox_serve_amd import block_attention as B
    n, hq, h, d, page = 6, 4, 2, 64, 16
    q, k, v = (torch.randn(n, x, d, device=dev, dtype=torch.bfloat16) for x in (hq, h, h))
    kv = torch.zeros(3, 2, page, h, d, dtype=torch.bfloat16, device=dev)
    pages, slots = torch.tensor([0, -1, 3, 1, 2, 2], device=dev), torch.tensor([15, 15, 15, -1, 16, 15], device=dev)
    out = torch.full((n, hq, d), 7.0, dtype=torch.bfloat16, device=dev)
    for n_req in (0, n):
        bounds, steps = B.new_bounds(kv, 16)
        B.rope_append(q, k, v, kv, None, torch.zeros(n, dtype=torch.int32, device=dev), pages, slots, bounds=bounds, steps=steps, out=out, n_req=n_req)
        assert torch.equal(out[[0, 5]], q[[0, 5]]) and (out[1:5] == 7).all()
        assert torch.equal(kv[[0, 2], 0, 15], k[[0, 5]]) and torch.equal(kv[[0, 2], 1, 15], v[[0, 5]])
        assert not kv[1].any() and not kv[:, :, :15].any()
        assert (steps[[0, 2]] > 0).all() and not steps[1].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_bounds_of_odd_keys(dev, d, block):
    """Zeros, subnormals, the type's largest and lowest, infinities and NaN; a channel of NaN; the same by update_bounds."""
    from vox_serve_amd import block_attention as B
    for dtype in (torch.bfloat16, torch.float16):
        s = Paged(dev, dtype, 3, d, 2 * block, [2 * block * 8], [1], seed=d + block, spare=0)
        k = s.kv[:, 0]
        k[0] = 0
        k[1, 3] = torch.finfo(dtype).max
        k[2, 5, 1, 7] = float("inf")
        k[2, 6, 1, 8] = float("-inf")
        k[3, 0, 2] = float("nan")
        k[4, :, 0, 9] = float("nan")
        k[5] *= 2.0 ** -20
        k[6, :, 1] = torch.finfo(dtype).smallest_normal / 4
        k[7, :block] = 127.0 * 0.5
        k[7, block:] = 1.0
        k[7, block + 1] = -2.0
        bounds, steps = B.new_bounds(s.kv, block)
        pages = torch.arange(8, device=dev).repeat_interleave(2)
        slots = torch.tensor([block - 1, 2 * block - 1], device=dev).repeat(8)
        B.update_bounds(s.kv, bounds, steps, pages, slots)
        want_b, want_s = s.bounds(block)
        assert torch.equal(bounds, want_b) and torch.equal(steps, want_s)


# ---------------------------------------------------------------- choose
SELECT = [  # heads, kv heads, dim, page, block, top, first, last, kv lengths, new rows
    (16, 8, 128, 128, 32, 8, 1, 2, [1000, 33, 600], [1, 1, 1]),
    (32, 2, 128, 64, 64, 5, 1, 2, [2000, 64, 320, 321], [1, 1, 1, 1]),
    (14, 2, 64, 48, 16, 9, 1, 2, [700, 150], [30, 21]),
    (8, 8, 64, 16, 16, 3, 0, 1, [300], [130]),
    (12, 4, 128, 32, 32, 7, 3, 4, [900, 260], [17, 3]),
    (64, 1, 64, 16, 16, 12, 2, 1, [500, 1], [2, 1]),
    (6, 2, 128, 128, 128, 4, 1, 1, [3000], [9]),
    (4, 2, 64, 16, 16, 70, 1, 2, [2100, 5], [3, 2]),        # more than a wave's lanes to take
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,h,d,page,block,top,first,last,kv_lens,q_lens", SELECT)
def test_select_blocks(dev, dtype, hq, h, d, page, block, top, first, last, kv_lens, q_lens):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, TYPES[dtype], h, d, page, kv_lens, q_lens, seed=top)
    q = s.rnd(s.n, hq, d)
    bounds, steps = s.bounds(block)
    nb, ns = bounds.cpu().numpy(), steps.cpu().numpy()
    want = np.stack([R.select(f64(q[i]), nb, ns, s.pages[s.req[i]], s.kvlen[i], block, top, first, last) for i in range(s.n)])
    for n_req in (0, len(q_lens)):
        for most in (max(kv_lens), 4 * max(kv_lens)):
            got = B.select_blocks(q, bounds, steps, *s.plan, block=block, top=top, max_kvlen=most, first=first, last=last, n_req=n_req)
            assert np.array_equal(got.cpu().numpy(), want)


def test_select_ties_zeros_and_odd_queries(dev):
    """Equal scores go to the older block; queries of zeros, NaN and infinities choose by the same rule."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 2, 64, 32, [32 * 40] * 6, [1] * 6, seed=4)
    s.kv[:, 0] = s.kv[:1, :1, :1, :, :][:, 0]                # every key the same
    q = s.rnd(6, 8, 64)
    q[1] = 0
    q[2, 3, 5] = float("nan")
    q[3, 0, 0] = float("inf")
    q[4] = float("nan")
    q[5, :4] *= 2.0 ** 100
    for mix in (False, True):
        if mix:
            s.kv[::3, 0] *= 2.0
        bounds, steps = s.bounds(32)
        nb, ns = bounds.cpu().numpy(), steps.cpu().numpy()
        want = np.stack([R.select(f64(q[i]), nb, ns, s.pages[i], s.kvlen[i], 32, 11, 1, 2) for i in range(6)])
        got = B.select_blocks(q, bounds, steps, *s.plan, block=32, top=11, max_kvlen=1280, n_req=6)
        assert np.array_equal(got.cpu().numpy(), want)
        if not mix:
            assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 38, 39]


def test_select_passes_rows_over_and_missing_pages(dev):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.float16, 2, 64, 16, [400, 400, 400], [1, 1, 1], seed=2)
    bounds, steps = s.bounds(16)
    q = s.rnd(5, 4, 64)
    req, lens = torch.tensor([0, 1, 2, 7, -1], device=dev), torch.tensor([400, 0, 400, 400, 400], device=dev)
    indices = s.indices.clone()
    indices[int(s.indptr[2]) + 3] = 10 ** 6
    indices[int(s.indptr[2]) + 9] = -5
    out = torch.full((5, 2, 6), 99, dtype=torch.int32, device=dev)
    B.select_blocks(q, bounds, steps, req, lens, s.indptr, indices, block=16, top=6, max_kvlen=400, out=out)
    pages = list(s.pages[2])
    pages[3], pages[9] = 10 ** 6, -5
    for i, p in ((0, s.pages[0]), (2, pages)):
        assert np.array_equal(out[i].cpu().numpy(), R.select(f64(q[i]), bounds.cpu().numpy(), steps.cpu().numpy(), p, 400, 16, 6, 1, 2))
    assert (out[[1, 3, 4]] == 99).all()
    # a row that claims more tokens than its request has pages, and one longer than max_kvlen says
    B.select_blocks(q[:2], bounds, steps, torch.tensor([2, 1], device=dev), torch.tensor([900, 400], device=dev), s.indptr, s.indices, block=16, top=6, max_kvlen=900, out=out[:2])
    assert np.array_equal(out[0].cpu().numpy(), R.select(f64(q[0]), bounds.cpu().numpy(), steps.cpu().numpy(), s.pages[2], 900, 16, 6, 1, 2))
    B.select_blocks(q[:2], bounds, steps, torch.tensor([2, 1], device=dev), torch.tensor([400, 400], device=dev), s.indptr, s.indices, block=16, top=6, max_kvlen=200, out=out[:2])
    assert np.array_equal(out[1].cpu().numpy(), R.select(f64(q[1]), bounds.cpu().numpy(), steps.cpu().numpy(), s.pages[1], 200, 16, 6, 1, 2))


# ---------------------------------------------------------------- attend
def check_attend(s, q, got, blocks, block, scale, rows=None):
    step = torch.finfo(s.dtype).eps / 2
    kv, lists = f64(s.kv), blocks.cpu().numpy()
    for i in rows if rows is not None else range(s.n):
        want, off = R.attend(f64(q[i]), kv, lists[i], s.pages[s.req[i]], s.kvlen[i], block, scale)
        far = np.abs(f64(got[i]) - want)
        assert (far <= step * np.abs(want) + off + torch.finfo(s.dtype).smallest_normal * step).all(), (i, float((far / (step * np.abs(want) + off + 1e-30)).max()))


def random_lists(s, h, block, top, seed):
    """Ascending lists of different lengths, empty ones among them."""
    r = np.random.default_rng(seed)
    out = np.full((s.n, h, top), -1, np.int32)
    for i, n in enumerate(s.kvlen):
        for g in range(h):
            have = -(-n // block)
            m = min(have, int(r.integers(0, top + 1)))
            out[i, g, :m] = np.sort(r.permutation(have)[:m])
    return torch.from_numpy(out).to(s.dev)


ATTEND = [  # heads, kv heads, dim, page, block, top, kv lengths, new rows
    (16, 8, 128, 128, 32, 8, [500, 33, 1, 256], [1, 1, 1, 1]),
    (32, 2, 128, 64, 64, 6, [700, 64, 65], [1, 1, 1]),
    (14, 2, 64, 48, 16, 9, [300, 120], [40, 23]),
    (8, 8, 64, 16, 16, 20, [400], [70]),
    (12, 4, 128, 32, 32, 7, [500, 90], [33, 5]),
    (64, 2, 64, 16, 16, 5, [100, 40], [7, 1]),
    (40, 1, 128, 32, 16, 12, [200, 90], [3, 1]),
    (6, 2, 128, 128, 128, 5, [1000], [19]),
    (4, 4, 64, 128, 128, 3, [130, 127, 129], [1, 2, 3]),
    (32, 2, 128, 256, 128, 40, [6000, 3000], [1, 1]),        # much to read for few rows
    (4, 2, 64, 16, 16, 130, [2500, 1800], [1, 1]),
    (10, 2, 128, 16, 16, 64, [900, 700], [50, 37]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,h,d,page,block,top,kv_lens,q_lens", ATTEND)
def test_block_attention(dev, dtype, hq, h, d, page, block, top, kv_lens, q_lens):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, TYPES[dtype], h, d, page, kv_lens, q_lens, seed=block + top)
    wide = s.rnd(s.n, (hq + 3) * d)
    q = wide[:, d:(hq + 1) * d].unflatten(1, (hq, d))         # rows apart
    blocks = random_lists(s, h, block, top, top)
    scale = d ** -0.5
    for n_req in (0, len(q_lens)):
        got = B.block_attention(q, s.kv, blocks, *s.plan, block=block, n_req=n_req)
        check_attend(s, q, got, blocks, block, scale)
    sharp = B.block_attention(q, s.kv, blocks, *s.plan, block=block, scale=1.0, n_req=len(q_lens))
    check_attend(s, q, sharp, blocks, block, 1.0)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [20, 9, 2]])
@pytest.mark.parametrize("hq,h,d", [(8, 2, 128), (16, 1, 64), (4, 2, 64)])
def test_attention_masked_places(dev, hq, h, d, q_lens):
    """NaN, infinities and the type's lowest value behind a row's last token, in blocks that it does not list, and in pages that are nobody's
    reach no row; where a row does see an infinity, its output is what the formula gives."""
    from vox_serve_amd import block_attention as B
    for dtype in (torch.bfloat16, torch.float16):
        s = Paged(dev, dtype, h, d, 32, [200, 90, 37], q_lens, seed=d)
        q = s.rnd(s.n, hq, d)
        blocks = random_lists(s, h, 16, 6, 5)
        want = B.block_attention(q, s.kv, blocks, *s.plan, block=16, n_req=3)
        check_attend(s, q, want, blocks, 16, d ** -0.5)
        # per request: tokens that none of its rows may see (behind the longest), then one row's own view of another's tokens
        bad = s.kv.clone()
        for fill in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
            b = bad.clone()
            owned = {p for pages in s.pages for p in pages}
            for p in range(b.shape[0]):
                if p not in owned:
                    b[p] = fill
            for r, n in enumerate(s.kv_lens):
                for t in range(n, len(s.pages[r]) * 32):
                    b[s.pages[r][t // 32], :, t % 32] = fill
            assert torch.equal(B.block_attention(q, b, blocks, *s.plan, block=16, n_req=3), want)
            # a request's newest token holds the fill: rows that see it feel it, the others do not
            b = s.kv.clone()
            n = s.kv_lens[0]
            b[s.pages[0][(n - 1) // 32], :, (n - 1) % 32] = fill
            got = B.block_attention(q, b, blocks, *s.plan, block=16, n_req=3)
            feel = torch.tensor([[s.req[i] == 0 and s.kvlen[i] == n and (n - 1) // 16 in blocks[i, g].tolist() for g in range(h)] for i in range(s.n)], device=dev)
            feel = feel.repeat_interleave(hq // h, 1)
            assert torch.equal(got[~feel], want[~feel])
            # a block that only one row lists
            if s.n > 6:
                lists = blocks.clone()
                lists[lists == 1] = 2
                lists[3, :, :] = -1
                lists[3, :, 0] = 1
                clean = B.block_attention(q, s.kv, lists, *s.plan, block=16, n_req=3)
                b = s.kv.clone()
                b[s.pages[0][0], :, 16:32] = fill
                got = B.block_attention(q, b, lists, *s.plan, block=16, n_req=3)
                others = [i for i in range(s.n) if i != 3]
                assert torch.equal(got[others], clean[others])


def test_attention_infinite_value_seen(dev):
    """One infinite value in a seen token: +inf in that channel, the others untouched; a NaN key poisons its row's heads only."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 2, 64, 32, [64], [8], seed=1)
    q = s.rnd(8, 4, 64)
    blocks = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev).repeat(8, 2, 1)
    clean = B.block_attention(q, s.kv, blocks, *s.plan, block=16, n_req=1)
    s.kv[s.pages[0][0], 1, 3, 0, 5] = float("inf")
    got = B.block_attention(q, s.kv, blocks, *s.plan, block=16, n_req=1)
    assert torch.isposinf(got[:, :2, 5]).all()
    keep = torch.ones(64, dtype=torch.bool)
    keep[5] = False
    assert torch.equal(got[:, :2, keep], clean[:, :2, keep]) and torch.equal(got[:, 2:], clean[:, 2:])
    s.kv[s.pages[0][1], 0, 28, 1, 0] = float("nan")          # token 60: seen by the last four rows
    got = B.block_attention(q, s.kv, blocks, *s.plan, block=16, n_req=1)
    assert torch.isnan(got[4:, 2:]).all() and torch.equal(got[:4, 2:], clean[:4, 2:])


def test_attention_entries_that_do_not_count(dev):
    """Equal and smaller entries, blocks behind the row, pages that do not exist: as if they were not listed; rows that see nothing stay."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.float16, 1, 64, 16, [100, 100, 100, 100], [1, 1, 1, 1], seed=3)
    q = s.rnd(6, 4, 64)
    odd = torch.tensor([[0, 0, 3, 3, 5, 2], [4, 1, 2, 5, 5, 6], [0, 2, 6, 7, 2000000000, 6], [-1, -1, 1, -1, 0, 2], [0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5]], dtype=torch.int32, device=dev)
    plain = torch.tensor([[0, 3, 5, -1, -1, -1], [4, 5, 6, -1, -1, -1], [0, 2, 6, -1, -1, -1], [1, 2, -1, -1, -1, -1]], dtype=torch.int32, device=dev)
    req, lens = torch.tensor([0, 1, 2, 3, 0, 9], device=dev), torch.tensor([100, 100, 100, 100, 0, 100], device=dev)
    for n_req in (0, 4, 6):
        out = torch.full((6, 4, 64), 5.0, dtype=torch.float16, device=dev)
        B.block_attention(q, s.kv, odd[:, None], req, lens, s.indptr, s.indices, block=16, n_req=n_req, out=out)
        assert (out[4:] == 5).all()
        check_attend(s, q, out, plain[:, None], 16, 0.125)
        indices = s.indices.clone()
        indices[0], indices[int(s.indptr[1]) + 4] = -1, 10 ** 8
        out = torch.empty_like(out)
        B.block_attention(q[:4], s.kv, plain[:, None], s.q_req, s.q_kvlen, s.indptr, indices, block=16, n_req=n_req, out=out[:4])
        few = torch.tensor([[3, 5, -1, -1, -1, -1], [5, 6, -1, -1, -1, -1], [0, 2, 6, -1, -1, -1], [1, 2, -1, -1, -1, -1]], dtype=torch.int32, device=dev)
        check_attend(s, q, out, few[:, None], 16, 0.125)
    empty = B.block_attention(q[:4], s.kv, torch.full((4, 1, 3), -1, device=dev), *s.plan, block=16)
    assert not empty.any()
    assert not B.block_attention(q[:4], s.kv, torch.empty(4, 1, 0, dtype=torch.int32, device=dev), *s.plan, block=16).any()
    assert B.block_attention(q[:0], s.kv, plain[:0, None], s.q_req[:0], s.q_kvlen[:0], s.indptr, s.indices, block=16).shape == (0, 4, 64)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0, 1e-12])
@pytest.mark.parametrize("q_lens", [[1, 1], [21, 6]])
def test_attention_scales(dev, scale, q_lens):
    """Negative, no and large scales; scores in rising order, so that the largest one moves again and again."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 2, 64, 32, [400, 90], q_lens, seed=3)
    for r, pages in enumerate(s.pages):
        for j, p in enumerate(pages):
            s.kv[p, 0] *= 0.2 * (j + 1)
    q = s.rnd(s.n, 8, 64)
    blocks = random_lists(s, 2, 16, 25, 4)
    check_attend(s, q, B.block_attention(q, s.kv, blocks, *s.plan, block=16, scale=scale, n_req=2), blocks, 16, scale)


def test_all_blocks_are_dense_attention(dev):
    from vox_serve_amd.flashinfer_utils import FlashInferPrefillWrapper
    hq, h, d, page, q_lens, kv_lens = 16, 8, 128, 32, [40, 1, 75], [140, 90, 75]
    need = [-(-n // page) for n in kv_lens]
    g = torch.Generator().manual_seed(8)
    kv = torch.randn(sum(need), 2, page, h, d, generator=g).bfloat16().to(dev)
    q = torch.randn(sum(q_lens), hq, d, generator=g).bfloat16().to(dev)
    w = FlashInferPrefillWrapper(None, hq, h, hq * d, page, device=dev)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)
    w.plan(i32([0, 40, 41, 116]), i32([0] + list(np.cumsum(need))), torch.randperm(sum(need), generator=g).int(), i32([n - (m - 1) * page for n, m in zip(kv_lens, need)]), torch.bfloat16)
    from vox_serve_amd import block_attention as B
    bounds, steps = B.new_bounds(kv, 16)
    blocks = w.select_blocks(q, bounds, steps, top=16)
    a, b = w.run_blocks(q, kv, blocks, 16).double(), w.run(q, kv).double()
    # both are within half a step of the same value, and fp32's share of it
    assert ((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -13).all()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_session(dev, dtype):
    """A prompt in two chunks and then decoded tokens: rotated and appended, blocks chosen, attended - every step against the oracle, on a cache
    and bounds that only these calls have written."""
    from vox_serve_amd import block_attention as B
    from vox_serve_amd.flashinfer_utils import FlashInferDecodeWrapper, FlashInferPrefillWrapper
    hq, h, d, page, block, top = 8, 2, 64, 32, 16, 6
    t, g = TYPES[dtype], torch.Generator().manual_seed(9)
    kv = torch.zeros(24, 2, page, h, d, dtype=t, device=dev)
    bounds, steps = B.new_bounds(kv, block)
    pages, have = [list(range(0, 12)), list(range(12, 24))], [0, 0]
    cs = table(dev, 512, d // 2)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)
    s = Paged(dev, t, h, d, page, [1, 1], [1, 1])

    def step(new, wrapper):
        for r in range(2):
            have[r] += new[r]
        need = [-(-n // page) for n in have]
        args = (i32([0] + list(np.cumsum(need))), i32([p for r in range(2) for p in pages[r][:need[r]]]), i32([n - (m - 1) * page for n, m in zip(have, need)]), t)
        if wrapper is FlashInferPrefillWrapper:
            args = (i32([0] + list(np.cumsum(new))),) + args
        w = wrapper(None, hq, h, hq * d, page, device=dev)
        w.plan(*args)
        rows = sum(new)
        qkv = torch.randn(rows, (hq + 2 * h) * d, generator=g).to(t).to(dev)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, h * d, h * d], 1))
        kvlen = [have[r] - new[r] + i + 1 for r in range(2) for i in range(new[r])]
        pos = torch.tensor(kvlen, device=dev) - 1
        qr = w.set_kv_cache_rope(kv, q, k, v, pos, cs, bounds=bounds, steps=steps)
        blocks = w.select_blocks(qr, bounds, steps, top)
        out = w.run_blocks(qr, kv, blocks, block)
        s.kv, s.req, s.kvlen, s.n, s.pages = kv, [r for r in range(2) for _ in range(new[r])], kvlen, rows, pages
        for r in range(2):                                    # every complete block's bounds are those of its keys
            for j in range(have[r] // block):
                p = pages[r][j * block // page]
                at = j * block % page
                for gh in range(h):
                    wb, ws = R.bounds(f64(kv[p, 0, at:at + block, gh]))
                    assert np.array_equal(bounds[p, gh, at // block].cpu().numpy(), wb) and float(steps[p, gh, at // block]) == ws
        nb, ns = bounds.cpu().numpy(), steps.cpu().numpy()
        for i in range(rows):
            assert np.array_equal(blocks[i].cpu().numpy(), R.select(f64(qr[i]), nb, ns, pages[s.req[i]], kvlen[i], block, top, 1, 2))
        check_attend(s, qr, out, blocks, block, d ** -0.5)

    step([70, 101], FlashInferPrefillWrapper)
    step([90, 13], FlashInferPrefillWrapper)
    for _ in range(20):
        step([1, 1], FlashInferDecodeWrapper)


@pytest.mark.parametrize("rows", [3, 64])
def test_captured_steps(dev, rows):
    """The three operators captured together, replayed with new inputs and eager calls of other sizes between: every replay is the eager result."""
    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    hq, h, d, page, block, top = 16, 8, 128, 64, 16, 12
    q_lens = [1] * 3 if rows == 3 else [60, 1, 3]
    s = Paged(dev, torch.bfloat16, h, d, page, [600, 333, 128], q_lens, seed=rows)
    qkv = s.rnd(s.n, (hq + 2 * h) * d)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, h * d, h * d], 1))
    pos, cs = s.q_kvlen - 1, table(dev, 1024, d // 2)
    bounds, steps = s.bounds(block)
    qr, blocks, out = torch.empty(s.n, hq, d, dtype=s.dtype, device=dev), torch.empty(s.n, h, top, dtype=torch.int32, device=dev), torch.empty(s.n, hq, d, dtype=s.dtype, device=dev)

    def calls(kv, b, st, qr, blocks, out):
        B.rope_append(q, k, v, kv, cs, pos, s.row_page, s.row_slot, bounds=b, steps=st, n_req=3, out=qr)
        B.select_blocks(qr, b, st, *s.plan, block=block, top=top, max_kvlen=600, n_req=3, out=blocks)
        B.block_attention(qr, kv, blocks, *s.plan, block=block, n_req=3, out=out)

    calls(s.kv, bounds, steps, qr, blocks, out)
    graphs = []
    for _ in range(2):
        with N.graph_capture() as cap:
            calls(s.kv, bounds, steps, qr, blocks, out)
        graphs.append(cap.graph)
    other = Paged(dev, torch.bfloat16, h, d, page, [2000], [1], seed=7)
    ob, os_ = other.bounds(block)
    oq = other.rnd(1, hq, d)
    for i in range(6):
        qkv.copy_(s.rnd(*qkv.shape))
        kv2, b2, s2 = s.kv.clone(), bounds.clone(), steps.clone()
        N.check(N.lib().vox_graph_launch(graphs[i % 2], N.stream()))
        got = [x.clone() for x in (qr, blocks, out, s.kv, bounds, steps)]
        B.block_attention(oq, other.kv, B.select_blocks(oq, ob, os_, *other.plan, block=block, top=100, max_kvlen=2000, n_req=1), *other.plan, block=block, n_req=1)
        want = [torch.empty_like(x) for x in (qr, blocks, out)]
        calls(kv2, b2, s2, *want)
        torch.cuda.synchronize()
        for x, y in zip(got, want + [kv2, b2, s2]):
            assert torch.equal(x, y)
    for gr in graphs:
        N.lib().vox_graph_destroy(gr)


def test_on_another_stream_and_two_at_once(dev):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 2, 128, 128, [9000, 9000], [1, 1], seed=6)
    q = s.rnd(2, 32, 128)
    bounds, steps = B.new_bounds(s.kv, 128)
    B.update_bounds(s.kv, bounds, steps, torch.arange(s.kv.shape[0], device=dev), torch.full((s.kv.shape[0],), 127, device=dev))
    want_b = B.select_blocks(q, bounds, steps, *s.plan, block=128, top=60, max_kvlen=9000, n_req=2)
    want = B.block_attention(q, s.kv, want_b, *s.plan, block=128, n_req=2)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                b = B.select_blocks(q, bounds, steps, *s.plan, block=128, top=60, max_kvlen=9000, n_req=2)
                got.append((b, B.block_attention(q, s.kv, b, *s.plan, block=128, n_req=2)))
    torch.cuda.synchronize()
    for b, o in got:
        assert torch.equal(b, want_b) and torch.equal(o, want)


def test_two_graphs_at_once(dev):
    """Two graphs of split calls, captured one behind the other and replayed on two streams beside eager calls: neither reaches the other's workspace."""
    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    sets = []
    for seed in (1, 2):
        s = Paged(dev, torch.bfloat16, 2, 128, 128, [9000, 9000], [1, 1], seed=seed)
        q, blocks = s.rnd(2, 32, 128), torch.arange(60, dtype=torch.int32, device=dev).repeat(2, 2, 1).contiguous()
        out = torch.empty_like(q)
        want = B.block_attention(q, s.kv, blocks, *s.plan, block=128, n_req=2)
        torch.cuda.synchronize()
        with N.graph_capture() as cap:
            B.block_attention(q, s.kv, blocks, *s.plan, block=128, n_req=2, out=out)
        sets.append((s, q, blocks, out, want, cap.graph, torch.cuda.Stream()))
    for _ in range(10):
        for s, q, blocks, out, want, graph, st in sets:
            with torch.cuda.stream(st):
                out.zero_()
                N.check(N.lib().vox_graph_launch(graph, N.stream()))
        eager = [B.block_attention(q, s.kv, blocks, *s.plan, block=128, n_req=2) for s, q, blocks, *_ in sets]
        torch.cuda.synchronize()
        for e, (_, _, _, out, want, *_) in zip(eager, sets):
            assert torch.equal(out, want) and torch.equal(e, want)
    for x in sets:
        N.lib().vox_graph_destroy(x[5])


def test_graph_keeps_what_its_calls_made(dev):
    """A run captured with int64 plans, q of heads that lie apart and results that only the next call takes: the graph's memory stays its own."""
    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    hq, h, d, block, top = 8, 2, 64, 16, 6
    s = Paged(dev, torch.bfloat16, h, d, 32, [700, 480], [1, 1], seed=8)
    bounds, steps = s.bounds(block)
    wide, k, v = s.rnd(2, hq, 2 * d), s.rnd(2, h, d), s.rnd(2, h, d)
    cs, plan = table(dev, 1024, d // 2), [x.long() for x in s.plan]
    where = (s.q_kvlen - 1).long(), s.row_page.long(), s.row_slot.long()

    def run():
        q = B.rope_append(wide[:, :, :d], k, v, s.kv, cs, *where, bounds=bounds, steps=steps, n_req=2)
        return B.block_attention(q, s.kv, B.select_blocks(q, bounds, steps, *plan, block=block, top=top, max_kvlen=700, n_req=2), *plan, block=block, n_req=2)

    want = run()
    torch.cuda.synchronize()
    with N.graph_capture() as cap:
        got = run()
    with torch.cuda.stream(N._capture_streams[torch.cuda.current_device()]):      # what this stream let go of would be handed out again here
        others = [torch.full((n,), 3, dtype=torch.int32, device=dev) for n in (2, 3, 12, 24, 100, 128, 512, 1024) for _ in range(8)]
    torch.cuda.synchronize()
    for _ in range(3):
        got.zero_()
        N.check(N.lib().vox_graph_launch(cap.graph, N.stream()))
        torch.cuda.synchronize()
        assert torch.equal(got, want) and all(bool((x == 3).all()) for x in others)
        for x in others:
            x.fill_(3)
    N.lib().vox_graph_destroy(cap.graph)


def test_results_do_not_depend_on_the_batch(dev):
    """The choice and the appended rows of a request are the same alone and among others."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 8, 128, 64, [3000, 1700, 900], [1, 1, 1], seed=12)
    q = s.rnd(3, 16, 128)
    bounds, steps = B.new_bounds(s.kv, 32)
    where = torch.arange(s.kv.shape[0], device=dev).repeat_interleave(2), torch.tensor([31, 63], device=dev).repeat(s.kv.shape[0])
    B.update_bounds(s.kv, bounds, steps, *where)
    every = B.select_blocks(q, bounds, steps, *s.plan, block=32, top=20, max_kvlen=3000, n_req=3)
    for i in range(3):
        one = B.select_blocks(q[i:i + 1], bounds, steps, s.q_req[i:i + 1], s.q_kvlen[i:i + 1], s.indptr, s.indices, block=32, top=20, max_kvlen=s.kvlen[i], n_req=1)
        assert torch.equal(one[0], every[i])


def test_offsets_beyond_32_bits(dev):
    """Pages whose elements lie more than 2^32 bytes, and 2^31 elements, behind the cache's start."""
    from vox_serve_amd import block_attention as B
    page, h, d = 128, 8, 128
    total = 2 ** 31 // (2 * page * h * d) + 9
    kv = torch.empty(total, 2, page, h, d, dtype=torch.bfloat16, device=dev)
    s = Paged(dev, torch.bfloat16, h, d, page, [128 * 8], [1], seed=5, spare=0)
    far = [total - 1 - i for i in range(8)]
    for i, p in enumerate(far):
        kv[p] = s.kv[s.pages[0][i]]
    small_b, small_s = B.new_bounds(s.kv, 16)
    slots = torch.arange(15, 128, 16, device=dev)
    B.update_bounds(s.kv, small_b, small_s, torch.tensor(s.pages[0], device=dev).repeat_interleave(8), slots.repeat(8))
    bounds, steps = B.new_bounds(kv, 16)
    B.update_bounds(kv, bounds, steps, torch.tensor(far, device=dev).repeat_interleave(8), slots.repeat(8))
    assert torch.equal(bounds[far], small_b[s.pages[0]]) and torch.equal(steps[far], small_s[s.pages[0]])
    q, indices = s.rnd(1, 16, d), torch.tensor(far, dtype=torch.int32, device=dev)
    want_b = B.select_blocks(q, small_b, small_s, *s.plan, block=16, top=20, max_kvlen=1024, n_req=1)
    got_b = B.select_blocks(q, bounds, steps, s.q_req, s.q_kvlen, s.indptr, indices, block=16, top=20, max_kvlen=1024, n_req=1)
    assert torch.equal(want_b, got_b)
    assert torch.equal(B.block_attention(q, s.kv, want_b, *s.plan, block=16, n_req=1), B.block_attention(q, kv, got_b, s.q_req, s.q_kvlen, s.indptr, indices, block=16, n_req=1))
    k = s.rnd(1, h, d)
    B.rope_append(q, k, k, kv, None, s.q_kvlen, torch.tensor([total - 1], device=dev), torch.tensor([100], device=dev))
    assert torch.equal(kv[total - 1, :, 100], k.expand(2, -1, -1))


# ---------------------------------------------------------------- every launch
def select_form(s, hq, block, top, most, n_req, first=1, last=2):
    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    return N.lib().vox_block_select_form(B._SELECT.pack(0, 16, 16, s.kv.shape[0], s.page, block, s.h, s.d, B._DTYPES[s.dtype], 16, 16, 16, 16, s.n, len(s.kv_lens), n_req, hq, most, 0, 16, 16, 0, 0, 0, top,
                                                        first, last))


def attend_form(s, hq, block, top, n_req):
    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    return N.lib().vox_block_attention_form(B._ATTEND.pack(16, 0, 0, s.kv.shape[0], s.page, block, s.h, s.d, B._DTYPES[s.dtype], 16, 16, 16, 16, s.n, len(s.kv_lens), n_req, hq, 2 ** 31 - 1, 0, 16, 16, 16,
                                                           0, 0, 0, top, 1.0))


def some(n, count, seed):
    """The first and last rows and some between."""
    r = np.random.default_rng(seed)
    return sorted(i for i in ({0, n - 1} if count < 3 else {0, 1, 15, 16, 17, n - 2, n - 1}) | set(int(x) for x in r.integers(0, n, count)) if 0 <= i < n)


SELECT_FORMS = [  # form, heads, kv heads, dim, page, block, top, kv lengths, new rows, max_kvlen
    (16, 16, 8, 128, 32, 16, 7, [300, 200, 90], [60, 30, 1], 300),
    (16, 28, 2, 64, 64, 32, 6, [2000], [601], 2000),
    (16, 8, 8, 64, 48, 16, 5, [400, 350], [90, 3], 16384),          # as many blocks as sixteen rows' keys may be
    (8, 16, 8, 128, 16, 16, 9, [280, 150], [85, 9], 16385),         # one more
    (8, 4, 4, 64, 128, 32, 20, [9000], [190], 40000),
    (8, 4, 4, 64, 128, 16, 33, [40000], [190], 40000),              # thousands of candidates
    (1, 4, 4, 64, 128, 16, 33, [300], [190], 65537),                # more than eight rows' keys may be
    (1, 8, 8, 128, 128, 16, 20, [9000, 700], [40, 1], 9000),
    (1, 4, 4, 64, 64, 64, 5, [640, 130], [1, 1], 640),
    (1, 16, 8, 128, 64, 16, 12, [9000, 8300], [17, 16], 9000),      # 513 to 4096 blocks, no CU left
    (1, 16, 8, 64, 128, 16, 12, [700, 40], [17, 16], 65536),
    (1, 16, 8, 64, 128, 16, 12, [66000, 40], [1, 32], 66000),       # more than 4096
    (-64, 4, 2, 128, 128, 16, 40, [20000, 16399], [1, 1], 524288),  # parts without a block among them
    (-5, 32, 2, 64, 128, 16, 17, [18000], [25], 18000),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("form,hq,h,d,page,block,top,kv_lens,q_lens,most", SELECT_FORMS)
def test_select_of_every_form(dev, dtype, form, hq, h, d, page, block, top, kv_lens, q_lens, most):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, TYPES[dtype], h, d, page, kv_lens, q_lens, seed=top)
    assert select_form(s, hq, block, top, most, len(q_lens)) == form
    q = s.rnd(s.n, hq, d)
    bounds, steps = B.new_bounds(s.kv, block)
    per = page // block
    B.update_bounds(s.kv, bounds, steps, torch.arange(s.kv.shape[0], device=dev).repeat_interleave(per), torch.arange(block - 1, page, block, device=dev).repeat(s.kv.shape[0]))
    # the cache's first page, by the oracle: the choice below is of these bounds
    for g in range(h):
        for j in range(per):
            wb, ws = R.bounds(f64(s.kv[0, 0, j * block:(j + 1) * block, g]))
            assert np.array_equal(bounds[0, g, j].cpu().numpy(), wb) and float(steps[0, g, j]) == ws
    got = B.select_blocks(q, bounds, steps, *s.plan, block=block, top=top, max_kvlen=most, n_req=len(q_lens)).cpu().numpy()
    nb, ns = bounds.cpu().numpy(), steps.cpu().numpy()
    long = max(kv_lens) // block > 500
    for i in some(s.n, 2 if long else 25, top):
        assert np.array_equal(got[i], R.select(f64(q[i]), nb, ns, s.pages[s.req[i]], s.kvlen[i], block, top, 1, 2)), i
    # every row's by another launch
    one = torch.cat([B.select_blocks(q[i:i + 1], bounds, steps, s.q_req[i:i + 1], s.q_kvlen[i:i + 1], s.indptr, s.indices, block=block, top=top, max_kvlen=max(kv_lens)) for i in range(s.n)])
    assert np.array_equal(got, one.cpu().numpy())


ATTEND_FORMS = [  # form, heads, kv heads, dim, page, block, top, kv lengths, new rows
    (16, 16, 8, 128, 32, 16, 6, [220, 150, 60], [180, 40, 9]),
    (16, 8, 8, 64, 16, 16, 5, [260, 100], [190, 35]),
    (8, 32, 8, 64, 64, 32, 4, [300, 64], [140, 20]),
    (10, 24, 8, 128, 128, 64, 3, [400], [190]),
    (4, 28, 4, 128, 48, 16, 7, [290], [260]),
    (2, 64, 4, 64, 32, 32, 4, [300, 33], [160, 33]),
    (2, 60, 4, 128, 16, 16, 9, [240], [200]),
    (1, 72, 4, 64, 16, 16, 5, [150], [140]),                # 18 heads on a kv head
    (16, 64, 32, 64, 32, 16, 4, [130, 60], [90, 60]),       # more tiles than CUs
    (16, 32, 32, 128, 16, 16, 4, [130, 60], [90, 60]),
    (16, 16, 8, 128, 16, 16, 200, [4000], [210]),           # lists that leave no room for eight waves' keys
    (-16, 16, 2, 128, 128, 128, 32, [5000, 4200], [1, 1]),
    (-3, 4, 4, 64, 64, 16, 100, [1700], [30]),
    (-64, 1, 1, 64, 128, 128, 128, [17000], [1]),
    (1, 4, 4, 128, 32, 32, 32, [1100], [30]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("form,hq,h,d,page,block,top,kv_lens,q_lens", ATTEND_FORMS)
def test_attention_of_every_form(dev, dtype, form, hq, h, d, page, block, top, kv_lens, q_lens):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, TYPES[dtype], h, d, page, kv_lens, q_lens, seed=block + top)
    assert attend_form(s, hq, block, top, len(q_lens)) == form
    q = s.rnd(s.n, hq, d)
    blocks = random_lists(s, h, block, top, top)
    got = B.block_attention(q, s.kv, blocks, *s.plan, block=block, n_req=len(q_lens))
    check_attend(s, q, got, blocks, block, d ** -0.5, some(s.n, 12, top))
    # all rows against the launch of a row each: both are within half a step, and fp32's share, of the same value
    other = B.block_attention(q, s.kv, blocks, *s.plan, block=block, n_req=0).double()
    a = got.double()
    step = torch.finfo(s.dtype).eps
    assert ((a - other).abs() <= step * torch.maximum(a.abs(), other.abs()) + 2.0 ** -13).all()
    # operands and results that lie on their type alone
    loose = torch.empty(s.n * hq * d + 3, dtype=s.dtype, device=dev)
    q2, out = loose[1:1 + s.n * hq * d].view(s.n, hq, d), torch.empty(s.n * hq * d + 1, dtype=s.dtype, device=dev)[1:].view(s.n, hq, d)
    q2.copy_(q)
    B.block_attention(q2, s.kv, blocks, *s.plan, block=block, n_req=len(q_lens), out=out)
    assert torch.equal(out, got)


@pytest.mark.parametrize("hq,h,d", [(16, 8, 128), (8, 8, 64), (28, 4, 64), (64, 32, 64)])
def test_rows_together_masked_places(dev, hq, h, d):
    """As test_attention_masked_places, where rows of a chunk share a launch's blocks: what one row may not see, or does not list, and another does, reaches the
    other alone, bit for bit."""
    from vox_serve_amd import block_attention as B
    for dtype in (torch.bfloat16, torch.float16):
        q_lens, kv_lens = [230, 40, 9], [300, 90, 37]
        s = Paged(dev, dtype, h, d, 32, kv_lens, q_lens, seed=d)
        assert attend_form(s, hq, 16, 6, 3) > 1
        q = s.rnd(s.n, hq, d)
        blocks = random_lists(s, h, 16, 6, 5)
        want = B.block_attention(q, s.kv, blocks, *s.plan, block=16, n_req=3)
        check_attend(s, q, want, blocks, 16, d ** -0.5, some(s.n, 8, d))
        lists = blocks.cpu().numpy()
        for fill in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
            b = s.kv.clone()
            owned = {p for pages in s.pages for p in pages}
            for p in range(b.shape[0]):
                if p not in owned:
                    b[p] = fill
            for r, n in enumerate(kv_lens):
                for t in range(n, len(s.pages[r]) * 32):
                    b[s.pages[r][t // 32], :, t % 32] = fill
            assert torch.equal(B.block_attention(q, b, blocks, *s.plan, block=16, n_req=3), want)
            # one token in the middle of the chunk
            token = 200
            b = s.kv.clone()
            b[s.pages[0][token // 32], :, token % 32] = fill
            got = B.block_attention(q, b, blocks, *s.plan, block=16, n_req=3)
            feel = np.array([[s.req[i] == 0 and s.kvlen[i] > token and token // 16 in lists[i, g].tolist() for g in range(h)] for i in range(s.n)])
            assert feel.any() and not feel.all()
            feel = torch.from_numpy(feel).to(dev).repeat_interleave(hq // h, 1)
            assert torch.equal(got[~feel], want[~feel])
            if fill != fill:
                assert torch.isnan(got[feel]).all()
        # an infinite value alone: that channel of the rows that see it, no other
        b = s.kv.clone()
        b[s.pages[0][token // 32], 1, token % 32, 0, 7] = float("inf")
        got = B.block_attention(q, b, blocks, *s.plan, block=16, n_req=3)
        feel = torch.tensor([s.req[i] == 0 and s.kvlen[i] > token and token // 16 in lists[i, 0].tolist() for i in range(s.n)], device=dev)
        g0 = hq // h
        assert torch.isposinf(got[feel][:, :g0, 7]).all()
        keep = torch.ones(d, dtype=torch.bool)
        keep[7] = False
        assert torch.equal(got[:, :, keep], want[:, :, keep]) and torch.equal(got[~feel], want[~feel]) and torch.equal(got[:, g0:], want[:, g0:])


def test_rows_together_entries_that_do_not_count(dev):
    """Lists that are not ascending, blocks far behind the sequence, pages that do not exist, rows that are passed over in the middle of others, in the launch of rows
    together; lists that lie thousands of blocks apart."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 8, 64, 16, [72000], [230], seed=3)
    hq = 16
    q = s.rnd(s.n, hq, 64)
    r = np.random.default_rng(1)
    lists = np.full((s.n, 8, 7), -1, np.int32)
    for i in range(s.n):
        for g in range(8):
            lists[i, g] = [0, 4499, 4498, 2 ** 31 - 1, 4499, 3, -7] if (i + g) % 3 == 0 else r.integers(-2, 4500, 7) if (i + g) % 3 == 1 else np.sort(r.permutation(4500)[:7])
    plain = np.full_like(lists, -1)
    for i in range(s.n):
        for g in range(8):
            seen, out = -1, []
            for j in lists[i, g].tolist():
                if j > seen:
                    seen = j
                    if j * 16 < s.kvlen[i]:
                        out.append(j)
            plain[i, g, :len(out)] = out
    lens, req = s.q_kvlen.clone(), s.q_req.clone()
    lens[5], lens[40], req[17], req[100] = 0, -3, -1, 1
    indices = s.indices.clone()
    indices[4499], indices[1000:1500] = -1, 10 ** 9
    plain[np.isin(plain, [4499] + list(range(1000, 1500)))] = -2        # (not listed)
    assert attend_form(s, hq, 16, 7, 1) == 16
    out = torch.full((s.n, hq, 64), 3.0, dtype=s.dtype, device=dev)
    B.block_attention(q, s.kv, torch.from_numpy(lists).to(dev), req, lens, s.indptr, indices, block=16, n_req=1, out=out)
    over = [5, 17, 40, 100]
    assert (out[over] == 3).all()
    rows = [i for i in some(s.n, 40, 2) if i not in over]
    ok = np.where(plain == -2, -1, plain)
    ok = np.stack([[np.concatenate([x[x >= 0], x[x < 0]]) for x in row] for row in ok])
    check_attend(s, q, out, torch.from_numpy(ok), 16, 0.125, rows)


def test_captured_rows_together(dev):
    """The launch of many rows captured beside selection and append, replayed with new inputs."""
    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    hq, h, d, page, block, top = 16, 8, 128, 64, 16, 12
    s = Paged(dev, torch.bfloat16, h, d, page, [600, 333, 128], [200, 31, 70], seed=4)
    assert attend_form(s, hq, block, top, 3) == 16 and select_form(s, hq, block, top, 600, 3) == 16
    qkv = s.rnd(s.n, (hq + 2 * h) * d)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, h * d, h * d], 1))
    pos, cs = s.q_kvlen - 1, table(dev, 1024, d // 2)
    bounds, steps = s.bounds(block)
    qr, blocks, out = torch.empty(s.n, hq, d, dtype=s.dtype, device=dev), torch.empty(s.n, h, top, dtype=torch.int32, device=dev), torch.empty(s.n, hq, d, dtype=s.dtype, device=dev)

    def calls(kv, b, st, qr, blocks, out):
        B.rope_append(q, k, v, kv, cs, pos, s.row_page, s.row_slot, bounds=b, steps=st, n_req=3, out=qr)
        B.select_blocks(qr, b, st, *s.plan, block=block, top=top, max_kvlen=600, n_req=3, out=blocks)
        B.block_attention(qr, kv, blocks, *s.plan, block=block, n_req=3, out=out)

    calls(s.kv, bounds, steps, qr, blocks, out)
    with N.graph_capture() as cap:
        calls(s.kv, bounds, steps, qr, blocks, out)
    for _ in range(4):
        qkv.copy_(s.rnd(*qkv.shape))
        kv2, b2, s2 = s.kv.clone(), bounds.clone(), steps.clone()
        N.check(N.lib().vox_graph_launch(cap.graph, N.stream()))
        got = [x.clone() for x in (qr, blocks, out, s.kv, bounds, steps)]
        want = [torch.empty_like(x) for x in (qr, blocks, out)]
        calls(kv2, b2, s2, *want)
        torch.cuda.synchronize()
        for x, y in zip(got, want + [kv2, b2, s2]):
            assert torch.equal(x, y)
    N.lib().vox_graph_destroy(cap.graph)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 240])
def test_many_small_weights(dev, dtype, rows):
    """One token with nearly all of the weight and 16 thousand with 2^-25 of it each: together they are more than a step of the output."""
    from vox_serve_amd import block_attention as B
    h, d, n = 8 if rows > 1 else 2, 64, 16384
    s = Paged(dev, TYPES[dtype], h, d, 128, [n], [rows], seed=rows)
    s.kv[:, 0] = 0
    s.kv[:, 1] = 1.0
    s.kv[s.pages[0][3], 0, 7] = 2.0
    s.kv[s.pages[0][3], 1, 7] = 0.0
    q = torch.full((rows, 2 * h, d), 1.0, dtype=s.dtype, device=dev)
    blocks = torch.arange(128, dtype=torch.int32, device=dev).repeat(rows, h, 1).contiguous()
    scale = 25 * np.log(2) / 128                              # the token's score is 25 log 2 above the others'
    assert (attend_form(s, 2 * h, 128, 128, 1) > 1) == (rows > 1)
    got = B.block_attention(q, s.kv, blocks, *s.plan, block=128, scale=float(scale), n_req=1)
    check_attend(s, q, got, blocks, 128, np.float32(scale).astype(np.float64), [0] if rows == 1 else [0, 100])
    assert (got > 4e-4).all()


def test_select_takes_nothing_but_the_ends(dev):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 8, 64, 16, [500, 320], [120, 1], seed=1)
    q = s.rnd(s.n, 16, 64)
    bounds, steps = s.bounds(16)
    for n_req in (0, 2):
        got = B.select_blocks(q, bounds, steps, *s.plan, block=16, top=5, first=2, last=3, max_kvlen=500, n_req=n_req)
        for i in range(s.n):
            have = -(-s.kvlen[i] // 16)
            assert (got[i].cpu() == torch.tensor([0, 1, have - 3, have - 2, have - 1])).all()
    # no row may see anything: nothing is written
    out = torch.full((s.n, 8, 5), 9, dtype=torch.int32, device=dev)
    B.select_blocks(q, bounds, steps, *s.plan, block=16, top=5, max_kvlen=0, out=out)
    assert (out == 9).all()


@pytest.mark.parametrize("alike", [0, 1, 5, 40])
@pytest.mark.parametrize("top", [4, 40, 70, 99, 130])
def test_rows_together_choose_among_many(dev, top, alike):
    """Few and many of 130 to 900 blocks, all different, all the same, or of a few kinds: what a wave narrows its search to fits its lanes or does not."""
    from vox_serve_amd import block_attention as B
    hq, h, d, block = 4, 4, 64, 16
    s = Paged(dev, torch.bfloat16, h, d, 32, [14400, 4500, 2150], [170, 30, 30], seed=top + alike)
    assert select_form(s, hq, block, top, 14400, 3) == 16
    if alike:                                                # every block of a page and a kind holds the same keys
        kinds = s.rnd(alike, h, d)
        s.kv[:, 0] = kinds[torch.arange(s.kv.shape[0], device=dev) % alike][:, None]
    q, (bounds, steps), pages = s.rnd(s.n, hq, d), B.new_bounds(s.kv, block), torch.arange(s.kv.shape[0], device=dev)
    B.update_bounds(s.kv, bounds, steps, pages.repeat_interleave(2), torch.tensor([15, 31], device=dev).repeat(s.kv.shape[0]))
    got = B.select_blocks(q, bounds, steps, *s.plan, block=block, top=top, max_kvlen=14400, n_req=3).cpu().numpy()
    nb, ns = bounds.cpu().numpy(), steps.cpu().numpy()
    for i in [0, 169, 170, 199, 200, 229]:
        assert np.array_equal(got[i], R.select(f64(q[i]), nb, ns, s.pages[s.req[i]], s.kvlen[i], block, top, 1, 2)), i
    one = torch.cat([B.select_blocks(q[i:i + 1], bounds, steps, s.q_req[i:i + 1], s.q_kvlen[i:i + 1], s.indptr, s.indices, block=block, top=top, max_kvlen=14400) for i in range(s.n)])
    assert np.array_equal(got, one.cpu().numpy())


def in_terms(p, n):
    """Weights as the sum of n bf16 terms."""
    out, left = np.zeros_like(p), p.copy()
    for _ in range(n):
        term = torch.from_numpy(left).to(torch.bfloat16).double().numpy()
        out, left = out + term, left - term
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,h,d,rows,top,form", [(16, 8, 128, 240, 3, 16), (8, 8, 64, 240, 3, 16), (4, 2, 128, 3, 3, 1), (32, 8, 64, 5, 3, 1), (4, 2, 128, 2, 100, -7)])
def test_weights_keep_their_bits(dev, dtype, hq, h, d, rows, top, form):
    """Three tokens of a block whose weighted values cancel to 2^-16 and less of themselves: what a softmax weight loses on its way into a product shows in the output, not below
    its rounding."""
    from vox_serve_amd import block_attention as B
    t, many = TYPES[dtype], 48 if top < 48 else 100
    s = Paged(dev, t, h, d, 64, [many * 16 + rows], [rows], seed=d + rows)
    assert attend_form(s, hq, 16, top, 1) == form
    g = torch.Generator().manual_seed(rows)
    as_type = lambda x: torch.from_numpy(x).to(t).double().numpy()
    z = as_type((2 * torch.rand(many, 16, h, generator=g, dtype=torch.float64) - 1).numpy())
    p, v = np.exp(z), np.zeros((many, 16, h, d))
    v[:, 3] = as_type((1 + torch.rand(many, h, d, generator=g, dtype=torch.float64)).numpy())
    v[:, 6] = as_type(-v[:, 3] * (p[:, 3] / p[:, 6])[..., None])
    v[:, 13] = as_type(-(v[:, 3] * p[:, 3, :, None] + v[:, 6] * p[:, 6, :, None]) / p[:, 13, :, None])
    s.kv.zero_()
    for j in range(many):
        page, at = s.pages[0][j // 4], j % 4 * 16
        s.kv[page, 0, at:at + 16, :, 0] = torch.from_numpy(z[j]).to(t).to(dev)
        s.kv[page, 1, at:at + 16] = torch.from_numpy(v[j]).to(t).to(dev)
    factor = 1 + np.arange(hq // h) / 64                     # the heads' q: what one of them cancels, the others of its kv head do not
    q = torch.zeros(rows, hq, d, dtype=t, device=dev)
    q[:, :, 0] = torch.from_numpy(np.tile(factor, h)).to(t).to(dev)
    lists = torch.full((rows, h, top), -1, dtype=torch.int32, device=dev)
    mine = [[i % many] if top < 48 else list(range(100)) for i in range(rows)]
    for i, m in enumerate(mine):
        lists[i, :, :len(m)] = torch.tensor(m, dtype=torch.int32, device=dev)
    got = f64(B.block_attention(q, s.kv, lists, *s.plan, block=16, scale=1.0, n_req=1)).reshape(rows, h, -1, d)
    half, seen = torch.finfo(t).eps / 2, False
    for i, m in enumerate(mine):
        w = np.exp(z[m][:, :, :, None] * factor)              # [blocks, 16, kv heads, heads of one]
        total = w.sum((0, 1))[..., None]
        want, size = (np.einsum("bthg,bthd->hgd", w, x) / total for x in (v[m], np.abs(v[m])))
        # A score is one product, exact.  A weight: its exponent's rounding, |z| log2 e < 4 (2^-23), log2 e's own (2^-24 of it, below 2^-23), the exponential's (2^-23) and
        # two fp16 terms' (2^-23; three of bf16 have all bits); three tokens of three terms, an addition each, 2^-23 where it cuts bits off; the parts' factors in
        # a list of many blocks are exponentials once more (2^-23 and its argument's, 2^-23), and its 3 x 100 tokens meet in sums of 32 that are added up (100 x 2^-23 of what
        # stands there, the blocks' own remainders).  The sum of the weights is in all of a column: (1600 + 64) 2^-23 of the output itself.
        rest = np.abs(np.einsum("bthg,bthd->bhgd", w, v[m]) / total).sum(0)
        tol = half * np.abs(want) + (13 if len(m) == 1 else 15) * 2.0 ** -23 * size + 1664 * 2.0 ** -23 * rest + torch.finfo(t).smallest_normal * half
        assert (np.abs(got[i] - want) <= tol).all(), (i, float((np.abs(got[i] - want) / tol).max()))
        if dtype == "bf16":
            seen |= bool((np.abs(np.einsum("bthg,bthd->hgd", in_terms(w, 2), v[m]) / total - want) > tol).any())
    assert seen or dtype != "bf16" or len(mine[0]) > 1       # two terms would be outside


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,h,d", [(16, 8, 128), (8, 8, 64), (28, 4, 64), (32, 8, 64)])
def test_rows_together_do_not_feel_each_others_keys(dev, dtype, hq, h, d):
    """Neighbouring rows that list neighbouring blocks: whatever scores one row's blocks give it, its neighbours' results stay as they are, bit for bit."""
    from vox_serve_amd import block_attention as B
    s = Paged(dev, TYPES[dtype], h, d, 32, [1300], [280], seed=d)
    lists = torch.tensor([[j for j in range(60) if not 16 <= j < 32 or j % 2 == i % 2] for i in range(s.n)], dtype=torch.int32, device=dev)[:, None].repeat(1, h, 1).contiguous()
    assert attend_form(s, hq, 16, lists.shape[2], 1) > 1
    q = s.rnd(s.n, hq, d)
    clean = B.block_attention(q, s.kv, lists, *s.plan, block=16, n_req=1)
    check_attend(s, q, clean, lists, 16, d ** -0.5, [0, 1, 17, 278, 279])
    for factor in (10.0, 100.0, -1000.0):
        kv = s.kv.clone()
        for j in range(16, 32, 2):
            kv[s.pages[0][j // 2], 0, :16] *= factor          # (an even block: the front half of its page)
        got = B.block_attention(q, kv, lists, *s.plan, block=16, n_req=1)
        assert torch.equal(got[1::2], clean[1::2])
        assert not torch.equal(got[::2], clean[::2])


def test_no_rows_with_long_lists(dev):
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 2, 64, 128, [300], [1])
    none, plan = s.rnd(1, 8, 64)[:0], (s.q_req[:0], s.q_kvlen[:0], s.indptr, s.indices)
    bounds, steps = B.new_bounds(s.kv, 128)
    before = s.kv.clone()
    for n_req in (0, 1):
        blocks = B.select_blocks(none, bounds, steps, *plan, block=128, top=1000, max_kvlen=300000, n_req=n_req)
        assert blocks.shape == (0, 2, 1000)
        assert B.block_attention(none, s.kv, blocks, *plan, block=128, n_req=n_req).shape == (0, 8, 64)
        empty = s.q_req[:0]
        assert B.rope_append(none, none[:, :2], none[:, :2], s.kv, None, empty, empty, empty, bounds=bounds, steps=steps, n_req=n_req).shape == (0, 8, 64)
    B.update_bounds(s.kv, bounds, steps, s.q_req[:0], s.q_req[:0])
    assert torch.equal(s.kv, before) and not bounds.any()


def choose_by_scores(q, bounds, steps, pages, n, block, top, first, last):
    """The oracle's choice with all of a row's scores at once: q [heads, dim], bounds [pages, kv heads, per, 2, dim] of whole numbers."""
    h, per, have = bounds.shape[1], bounds.shape[2], -(-n // block)
    j = np.arange(first, have - last)
    page, out = np.asarray(pages)[j // per], np.zeros((h, top), np.int64)
    for g in range(h):
        mine = q[g * (q.shape[0] // h):(g + 1) * (q.shape[0] // h)]
        a = np.clip(np.rint(mine / R.step_of(mine)), -127, 127).astype(np.int64)
        b = bounds[page, g, j % per].astype(np.int64)
        whole = sum(np.maximum(row * b[:, 0], row * b[:, 1]).sum(1) for row in a)
        score = whole.astype(np.float32) * steps[page, g, j % per]
        best = j[np.argsort(-score, kind="stable")[:top - first - last]]
        out[g] = np.sort(np.concatenate([np.arange(first), best, np.arange(have - last, have)]))
    return out


@pytest.mark.parametrize("kinds", [0, 1, 9])
@pytest.mark.parametrize("lens,rows,form", [
    # blocks of 16 tokens; a row alone in parts, whose choice has up to 2, 4, 8 and 32 keys a lane
    ([1500], 1, -6), ([2051], 1, -9), ([2052], 1, -9), ([4099], 1, -17), ([4100], 1, -17), ([6000], 1, -24), ([8195], 1, -33), ([8196], 1, -33), ([20001], 1, -79), ([32768], 1, -128),
    # eight waves a row: 2, 4 and 8 keys a lane
    ([900, 1027, 1028, 2051, 2052, 3333, 4096], 70, 1),
    # sixteen: 2, 4, 8, 16 and 32
    ([700, 2051, 2052, 4099, 4100, 8195, 8196, 16387, 16388, 25000, 32768], 66, 1),
    # rows of a chunk together, a wave a row: 2 to 16 of up to 1024 blocks, 2 to 64 of up to 4096
    ([35, 131, 132, 259, 260, 515, 516, 1024], 330, 16), ([40, 131, 132, 260, 515, 516, 1027, 1028, 2051, 2052, 4096], 330, 8),
])
def test_select_among_many_thousands(dev, kinds, lens, rows, form):
    """Each number of keys a lane that a choice has, at its borders, with all scores different, all the same, and of a few kinds: equal ones on both sides of waves."""
    from vox_serve_amd import block_attention as B
    from vox_serve_amd import _native as N
    hq, h, d, block, per, top = 4, 2, 64, 16, 8, 29
    g = np.random.default_rng(sum(lens) + kinds)
    most = max(lens)
    pages = -(-most // per) if not kinds else kinds
    b = np.sort(g.integers(-127, 128, (pages, h, per, 2, d)), axis=3)[..., ::-1, :].astype(np.int8)
    st = (2.0 ** g.integers(-3, 2, (pages, h, per))).astype(np.float32)
    if kinds:
        b[:], st[:] = b[:, :, :1], st[:, :, :1]
    table_ = g.permutation(pages) if not kinds else g.integers(0, pages, -(-most // per))
    blocks = [lens[i % len(lens)] for i in range(rows)]
    kvlen = [n * block - int(x) for n, x in zip(blocks, g.integers(0, block, rows))]
    q = torch.from_numpy(g.standard_normal((rows, hq, d))).to(torch.bfloat16).to(dev)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)
    bounds, steps = torch.from_numpy(b.copy()).to(dev), torch.from_numpy(st).to(dev)
    args, n_req = (i32([0] * rows), i32(kvlen), i32([0, len(table_)]), i32(table_)), 1 if form > 1 else rows
    sizes = B._SELECT.pack(0, 16, 16, pages, per * block, block, h, d, 0, 16, 16, 16, 16, rows, 1, n_req, hq, max(kvlen), 0, 16, 16, 0, 0, 0, top, 1, 2)
    assert N.lib().vox_block_select_form(sizes) == form
    got = B.select_blocks(q, bounds, steps, *args, block=block, top=top, max_kvlen=max(kvlen), n_req=n_req).cpu().numpy()
    for i in range(min(rows, 2 * len(lens))):
        assert np.array_equal(got[i], choose_by_scores(f64(q[i]), b, st, table_, kvlen[i], block, top, 1, 2)), (i, kvlen[i])
    small = min(range(rows), key=lambda i: kvlen[i])
    if blocks[small] < 3000:
        assert np.array_equal(got[small], R.select(f64(q[small]), b, st, table_.tolist(), kvlen[small], block, top, 1, 2))


def test_graphs_give_their_memory_back(dev):
    """Captured, replayed and destroyed again and again: what is allocated stays what it was; so does it behind a body that raises, and for eager calls during a capture."""
    import threading

    from vox_serve_amd import _native as N
    from vox_serve_amd import block_attention as B
    s = Paged(dev, torch.bfloat16, 2, 128, 128, [9000, 9000], [1, 1], seed=6)
    q, plan = s.rnd(2, 32, 256)[:, :, :128], [x.long() for x in s.plan]
    bounds, steps = B.new_bounds(s.kv, 128)
    B.update_bounds(s.kv, bounds, steps, torch.arange(s.kv.shape[0], device=dev), torch.full((s.kv.shape[0],), 127, device=dev))

    def run():
        return B.block_attention(q, s.kv, B.select_blocks(q, bounds, steps, *plan, block=128, top=60, max_kvlen=9000, n_req=2), *plan, block=128, n_req=2)

    want, sizes = run(), []
    for i in range(8):
        with N.graph_capture() as cap:
            got = run()
        assert N._graph_memory[cap.graph.value]
        for _ in range(3):
            got.zero_()
            N.check(N.lib().vox_graph_launch(cap.graph, N.stream()))
            assert torch.equal(got, want)
        # a body that raises behind its calls
        with pytest.raises(KeyError):
            with N.graph_capture() as failed:
                run()
                raise KeyError(i)
        assert not failed.held
        N.lib().vox_graph_destroy(cap.graph)
        assert not N._graph_memory and not N._capturing
        del got, cap, failed
        torch.cuda.synchronize()
        sizes.append(torch.cuda.memory_allocated())
    assert len(set(sizes)) == 1
    # another thread's eager calls while this one captures, and a stream forked from the capture
    done, side = [], torch.cuda.Stream()

    def other():
        with torch.cuda.device(dev), torch.cuda.stream(torch.cuda.Stream()):
            done.append(run())
            torch.cuda.current_stream().synchronize()

    with N.graph_capture() as cap:
        first = run()
        held = len(cap.held)
        worker = threading.Thread(target=other)
        worker.start()
        worker.join()
        assert len(cap.held) == held and torch.is_tensor(done[0])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = run()
        torch.cuda.current_stream().wait_stream(side)
        assert len(cap.held) == 2 * held
    assert torch.equal(done[0], want)
    for _ in range(3):
        first.zero_(), second.zero_()
        N.check(N.lib().vox_graph_launch(cap.graph, N.stream()))
        assert torch.equal(first, want) and torch.equal(second, want)
    N.lib().vox_graph_destroy(cap.graph)


def test_rope_append_far_positions(dev):
    """Positions behind apply_rope_pos_ids' own 8192, by a table of the caller's length; behind that one's end its last row."""
    from vox_serve_amd.flashinfer_utils import FlashInferDecodeWrapper, apply_rope_pos_ids, rope_table
    hq, h, d, page, kv_lens = 8, 2, 64, 128, [5000, 131072, 9000]
    need = [-(-n // page) for n in kv_lens]
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(3, x, d, generator=g).bfloat16().to(dev) for x in (hq, h, h))
    kv = torch.zeros(sum(need), 2, page, h, d, dtype=torch.bfloat16, device=dev)
    w = FlashInferDecodeWrapper(None, hq, h, hq * d, page, device=dev)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)
    w.plan(i32([0] + list(np.cumsum(need))), torch.randperm(sum(need), generator=g).int(), i32([n - (m - 1) * page for n, m in zip(kv_lens, need)]), torch.bfloat16)
    cs = rope_table(131072, d, rope_theta=1e6, device=dev)
    for pos in (torch.tensor(kv_lens, device=dev) - 1, torch.tensor([8191, 8192, 200000], device=dev)):
        got = w.set_kv_cache_rope(kv, q, k, v, pos, cs)
        want = R.rotate(f64(q), cs.cpu().numpy(), pos.cpu().numpy(), False)
        assert (np.abs(f64(got) - want) <= 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -8) + 2.0 ** -22 * np.abs(f64(q)).max(-1, keepdims=True)).all()
        near = pos < 8192
        qr, kr = apply_rope_pos_ids(q, k, pos, rope_theta=1e6)
        assert torch.equal(got[near], qr[near]) and torch.equal(kv[w._meta["page"].long(), 0, w._meta["slot"].long()][near], kr[near])
        assert not torch.equal(got[~near], qr[~near])


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -110, -(2.0 ** -104), 1e38])
@pytest.mark.parametrize("rows", [1, 240])
def test_attention_scales_of_all_sizes(dev, rows, scale):
    """Scores of 2^105 under no scale, under scales that bring them to about one, and scores of 2^-117 under the largest one: what the formula gives."""
    from vox_serve_amd import block_attention as B
    h, d = 8, 64
    s = Paged(dev, torch.bfloat16, h, d, 32, [400], [rows], seed=rows)
    q = s.rnd(rows, 2 * h, d)
    if abs(scale) < 1:                                       # (powers of two: exact)
        q *= 2.0 ** 52
        s.kv[:, 0] *= 2.0 ** 50
    else:
        q *= 2.0 ** -60
        s.kv[:, 0] *= 2.0 ** -60
    blocks = torch.arange(10, dtype=torch.int32, device=dev).repeat(rows, h, 1).contiguous()
    assert (attend_form(s, 2 * h, 16, 10, 1) > 1) == (rows > 1)
    got = B.block_attention(q, s.kv, blocks, *s.plan, block=16, scale=scale, n_req=1)
    check_attend(s, q, got, blocks, 16, float(np.float32(scale)), [0] if rows == 1 else [0, 100, 239])


def test_threads_at_once(dev):
    """Calls of several threads, each on its own stream: the same kernels with more and less LDS, parts and none."""
    import threading

    from vox_serve_amd import block_attention as B
    h, d, hq = 2, 128, 32
    s = Paged(dev, torch.bfloat16, h, d, 128, [70000, 70000], [1, 1], seed=3)
    q = s.rnd(2, hq, d)
    bounds, steps = B.new_bounds(s.kv, 16)
    pages = torch.arange(s.kv.shape[0], device=dev).repeat_interleave(8)
    B.update_bounds(s.kv, bounds, steps, pages, torch.arange(15, 128, 16, device=dev).repeat(s.kv.shape[0]))

    def run(top, rows):
        qs, req = q.repeat(rows, 1, 1), s.q_req.repeat(rows)
        lens = torch.minimum(s.q_kvlen.repeat(rows), torch.full((2 * rows,), 1000 * top, dtype=torch.int32, device=dev))
        most = min(70000, 1000 * top)
        b = B.select_blocks(qs, bounds, steps, req, lens, s.indptr, s.indices, block=16, top=top, max_kvlen=most)
        return b, B.block_attention(qs, s.kv, b, req, lens, s.indptr, s.indices, block=16)

    kinds = [(10, 80), (70, 1), (66, 70), (400, 1), (1000, 3), (62, 66)]
    want = [run(*k) for k in kinds]
    torch.cuda.synchronize()
    errors = []

    def loop(first):
        try:
            with torch.cuda.device(dev), torch.cuda.stream(torch.cuda.Stream()):
                for i in range(40):
                    k = (first + i) % len(kinds)
                    got = run(*kinds[k])
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(got[0], want[k][0]) and torch.equal(got[1], want[k][1]), kinds[k]
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 1e4])
@pytest.mark.parametrize("hq,h,d,rows,top", [(16, 8, 128, 230, 30), (8, 8, 64, 230, 30), (12, 4, 64, 3, 30), (32, 2, 128, 1, 120), (40, 1, 64, 2, 40)])
def test_queries_of_others_change_nothing(dev, hq, h, d, rows, top, fill):
    """A row's, and a head's, results are the same bits whatever queries the others have: NaN and infinities that send their tile through the second pass, scores that are large."""
    from vox_serve_amd import block_attention as B
    for dtype in (torch.bfloat16, torch.float16):
        s = Paged(dev, dtype, h, d, 32, [2000], [rows], seed=top)
        q, blocks = s.rnd(rows, hq, d), random_lists(s, h, 16, top, 3)
        blocks[0, :, :] = torch.arange(top, dtype=torch.int32, device=dev)
        clean = B.block_attention(q, s.kv, blocks, *s.plan, block=16, n_req=1)
        bad = torch.zeros(rows, hq, dtype=torch.bool, device=dev)
        bad[::3, ::2] = True
        q2 = q.clone()
        q2[bad] *= fill
        got = B.block_attention(q2, s.kv, blocks, *s.plan, block=16, n_req=1)
        assert torch.equal(got[~bad], clean[~bad])
        seen = (blocks >= 0).any(-1).repeat_interleave(hq // h, 1) & bad
        assert seen.any() and (torch.isnan(got[seen]).any(-1).all() if not fill < 1e9 else not torch.equal(got[seen], clean[seen]))
