"""What block_attention refuses, before anything reaches a GPU: by the C entry points (the argument structs with one field wrong at a time) and by the
Python functions; and that the packed structs are the header's."""
import os
import shutil
import subprocess

import pytest
import torch

from vox_serve_amd import _native as N
from vox_serve_amd import block_attention as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 4096           # an address for the checks to look at; nothing reads it
CACHE = dict(kv=AT, bounds=AT, steps=AT, n_pages=4, page_size=128, block=32, kv_heads=2, head_dim=128, dtype=0)
ROWS = dict(q_req=AT, q_kvlen=AT, kv_indptr=AT, kv_indices=AT, n_rows=3, n_req=2, n_own=0, heads=16, max_kvlen=400, pad=0)
APPEND = dict(CACHE, q=AT, k=AT, v=AT, q_out=AT, pos=AT, page=AT, slot=AT, table=AT, q_stride=2048, k_stride=256, v_stride=256, n_rows=3, n_own=0, heads=16, rot=128,
              interleave=0, table_max_pos=100)
SELECT = dict(CACHE, **ROWS, q=AT, blocks=AT, workspace=AT, workspace_bytes=1 << 40, q_stride=2048, top=8, first=1, last=2)
ATTEND = dict(CACHE, **ROWS, q=AT, blocks=AT, out=AT, workspace=AT, workspace_bytes=1 << 40, q_stride=2048, top=8, scale=0.1)


def call(fn, packer, fields, **wrong):
    return getattr(N.lib(), fn)(None, None, packer.pack(*dict(fields, **wrong).values()))


BAD_CACHE = [dict(kv=0), dict(kv=AT + 8), dict(n_pages=0), dict(page_size=0), dict(kv_heads=0), dict(kv_heads=-2), dict(dtype=2), dict(block=8), dict(block=0), dict(block=96),
             dict(page_size=100), dict(page_size=16), dict(head_dim=96), dict(head_dim=0)]
BAD_BOUNDS = [dict(steps=0), dict(bounds=AT + 4), dict(steps=AT + 2)]
BAD_ROWS = [dict(n_rows=-1), dict(n_req=-1), dict(n_own=-1), dict(heads=0), dict(heads=15), dict(heads=130), dict(max_kvlen=-1), dict(q_req=0), dict(q_kvlen=0), dict(kv_indptr=0),
            dict(kv_indices=0), dict(q=0), dict(q=AT + 1), dict(q_stride=-1), dict(blocks=0)]


@pytest.mark.parametrize("wrong", BAD_CACHE + BAD_BOUNDS + [dict(q=0), dict(k=0), dict(v=0), dict(q_out=0), dict(page=0), dict(slot=0), dict(pos=0), dict(table=0), dict(table=AT + 2),
                                                             dict(table_max_pos=0), dict(rot=130), dict(rot=3), dict(rot=-2), dict(n_rows=-1), dict(n_own=-1), dict(heads=0), dict(q=AT + 1),
                                                             dict(q_stride=-5), dict(head_dim=127, bounds=0), dict(head_dim=514, bounds=0)], ids=str)
def test_rope_append_refuses(wrong):
    assert call("vox_rope_append", B._APPEND, APPEND, **wrong) == 1
    assert b"rope_append" in N.lib().vox_last_error()


@pytest.mark.parametrize("wrong", BAD_BOUNDS + BAD_ROWS + [w for w in BAD_CACHE if "kv" not in w]
                         + [dict(bounds=0), dict(top=2), dict(top=1025), dict(first=-1), dict(last=0), dict(first=7), dict(first=2 ** 31 - 1), dict(max_kvlen=32 * 32768 + 1)], ids=str)
def test_block_select_refuses(wrong):
    assert call("vox_block_select", B._SELECT, SELECT, **wrong) == 1
    assert b"block_select" in N.lib().vox_last_error()


@pytest.mark.parametrize("wrong", BAD_CACHE + BAD_ROWS + [dict(out=0), dict(out=AT + 1), dict(top=-1), dict(top=1025), dict(scale=float("inf")),
                                                               dict(scale=float("nan"))], ids=str)
def test_block_attention_refuses(wrong):
    assert call("vox_block_attention", B._ATTEND, ATTEND, **wrong) == 1
    assert b"block_attention" in N.lib().vox_last_error()


@pytest.mark.parametrize("wrong", BAD_CACHE + BAD_BOUNDS + [dict(bounds=0)], ids=str)
def test_block_bounds_refuses(wrong):
    fields = B._BOUNDS.pack(*dict(CACHE, **wrong).values())
    assert N.lib().vox_block_bounds(None, None, fields, AT, AT, 3) == 1
    assert b"block_bounds" in N.lib().vox_last_error()


def test_missing_arguments_and_nothing_to_do():
    L = N.lib()
    for fn in ("vox_rope_append", "vox_block_select", "vox_block_attention"):
        assert getattr(L, fn)(None, None, None) == 1
    assert L.vox_block_bounds(None, None, None, AT, AT, 1) == 1
    assert L.vox_block_bounds(None, None, B._BOUNDS.pack(*CACHE.values()), None, AT, 1) == 1
    assert L.vox_block_bounds(None, None, B._BOUNDS.pack(*CACHE.values()), AT, AT, -1) == 1
    assert L.vox_block_select_workspace_bytes(B._SELECT.pack(*dict(SELECT, top=2).values())) == -1
    assert L.vox_block_attention_workspace_bytes(B._ATTEND.pack(*dict(ATTEND, top=-1).values())) == -1
    # no rows: done, and no pointer is asked for
    assert call("vox_rope_append", B._APPEND, APPEND, n_rows=0, q=0, k=0, v=0, page=0) == 0
    assert call("vox_block_select", B._SELECT, SELECT, n_rows=0, q=0, q_req=0) == 0
    assert call("vox_block_attention", B._ATTEND, ATTEND, n_rows=0, q=0, out=0, q_req=0) == 0
    assert L.vox_block_bounds(None, None, B._BOUNDS.pack(*CACHE.values()), None, None, 0) == 0


def test_packed_structs_are_the_headers(tmp_path):
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include "voxhip.h"\n#include <stdio.h>\n#include <stddef.h>\n#define P(t, f) printf("%zu ", offsetof(t, f))\n#define Z(t) printf("%zu\\n", sizeof(t))\nint main(void) {\n'
                   + "".join(f"P({t}, {f});" for t, f in (("vox_rope_append_args", "q_stride"), ("vox_rope_append_args", "table_max_pos"))) + "Z(vox_rope_append_args);"
                   + "P(vox_block_cache, dtype); Z(vox_block_cache);"
                   + "".join(f"P(vox_block_select_args, {f});" for f in ("rows.max_kvlen", "q", "q_stride", "last")) + "Z(vox_block_select_args);"
                   + "".join(f"P(vox_block_attention_args, {f});" for f in ("rows.heads", "out", "top", "scale")) + "Z(vox_block_attention_args);\nreturn 0;\n}\n")
    subprocess.check_call([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    lines = [[int(x) for x in line.split()] for line in subprocess.check_output([str(tmp_path / "s")], text=True).splitlines()]

    def at(packer, fields, *names):
        """Where a field's bytes lie: what changes when it does."""
        out = []
        for n in names:
            a, b = (packer.pack(*dict(fields, **{n: v}).values()) for v in ((1, 2) if n != "scale" else (1.0, -1.0)))
            out.append(min(i for i in range(len(a)) if a[i] != b[i]) // 4 * 4)
        return out + [packer.size]

    assert lines == [at(B._APPEND, APPEND, "q_stride", "table_max_pos"), at(B._BOUNDS, CACHE, "dtype"), at(B._SELECT, SELECT, "max_kvlen", "q", "q_stride", "last"),
                     at(B._ATTEND, ATTEND, "heads", "out", "top", "scale")]


def test_python_functions_refuse():
    """Shapes, types and places, on the CPU; the C entry points' own refusals come behind these."""
    kv = torch.zeros(2, 2, 32, 2, 64, dtype=torch.bfloat16)
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    one = torch.zeros(3, dtype=torch.int32)
    bounds, steps = B.new_bounds(kv, 16)
    assert bounds.shape == (2, 2, 2, 2, 64) and bounds.dtype is torch.int8 and steps.shape == (2, 2, 2)
    with pytest.raises(ValueError, match="whole blocks"):
        B.new_bounds(kv, 24)
    with pytest.raises(ValueError, match="HIP device"):
        B.rope_append(q, k, k, kv, None, one, one, one)
    with pytest.raises(ValueError, match="HIP device"):
        B.block_attention(q, kv, torch.zeros(3, 2, 2, dtype=torch.int32), one, one, one, one, block=16)
    with pytest.raises(ValueError, match="HIP device"):
        B.select_blocks(q, bounds, steps, one, one, one, one, block=16, top=4, max_kvlen=32)
    with pytest.raises(ValueError, match="HIP device"):
        B.update_bounds(kv, bounds, steps, one, one)
    with pytest.raises(ValueError, match="kv_cache has shape"):
        B.rope_append(q, k, k, kv[:, :1], None, one, one, one)
    with pytest.raises(ValueError, match="kv_cache has shape"):
        B.update_bounds(kv.transpose(2, 3), bounds, steps, one, one)
    with pytest.raises(TypeError, match="kv_cache is"):
        B.block_attention(q, kv.float(), torch.zeros(3, 2, 2, dtype=torch.int32), one, one, one, one, block=16)
    # the checks behind the device's, on their own
    with pytest.raises(ValueError, match="pages has shape"):
        B._ints(one, (4,), one.device, "pages")
    with pytest.raises(TypeError, match="int32 or int64"):
        B._ints(one.float(), (3,), one.device, "pages")
    assert B._ints(one.long(), (3,), one.device, "pages").dtype is torch.int32
    with pytest.raises(ValueError, match="q has shape"):
        B._heads(q, 3, 128, kv, "q")
    with pytest.raises(ValueError, match="q is torch.float16"):
        B._heads(q.half(), 3, 64, kv, "q")
    assert B._heads(q.transpose(0, 1).contiguous().transpose(0, 1), 3, 64, kv, "q").is_contiguous()       # heads apart: laid together
    wide = torch.zeros(3, 512, dtype=torch.bfloat16)[:, 64:320].unflatten(1, (4, 64))
    assert B._heads(wide, 3, 64, kv, "q") is wide                                                          # rows apart: taken as they are
    with pytest.raises(ValueError, match="not those of a cache"):
        B._bounds_of(kv, bounds[:1].contiguous(), steps[:1].contiguous())
    with pytest.raises(ValueError, match="steps is"):
        B._bounds_of(kv, bounds, steps.double())
    with pytest.raises(ValueError, match="bounds is"):
        B._bounds_of(kv, bounds.int(), steps)
    with pytest.raises(ValueError, match="out is"):
        B._out(torch.zeros(3, 4, 64), q.shape, torch.bfloat16, q.device)


def test_bounds_and_steps_come_together():
    kv = torch.zeros(2, 2, 32, 2, 64, dtype=torch.bfloat16)
    bounds, steps = B.new_bounds(kv, 16)
    for pair in ((bounds, None), (None, steps)):
        with pytest.raises(ValueError, match="come together"):
            B._bounds_of(kv, *pair)


@pytest.mark.parametrize("rows,own", [(0, 0), (0, 3), (3, 0)])
@pytest.mark.parametrize("top,block", [(8, 16), (16, 128), (1024, 128), (0, 16)])
def test_sizes_without_rows(rows, own, top, block):
    """What a call of no rows asks for: no workspace, a launch of some kind - and an answer, whatever its lists' length."""
    L, wrong = N.lib(), dict(n_rows=rows, n_own=own, top=top, block=block, page_size=256)
    attend, select = (B._ATTEND.pack(*dict(ATTEND, **wrong).values()), B._SELECT.pack(*dict(SELECT, **dict(wrong, top=max(top, 3)), max_kvlen=400).values()))
    long = B._SELECT.pack(*dict(SELECT, **dict(wrong, top=max(top, 3)), max_kvlen=16 * 5000).values())
    assert L.vox_block_attention_form(attend) != 0 and L.vox_block_select_form(select) != 0 and L.vox_block_select_form(long) != 0
    for room in (L.vox_block_attention_workspace_bytes(attend), L.vox_block_select_workspace_bytes(select), L.vox_block_select_workspace_bytes(long)):
        assert room == 0 if rows == 0 else room >= 0
    assert B._attend_room(rows, own, 16, 2, 128, 0, 256, block, top) >= 0


def test_graph_memory_goes_with_its_graph(monkeypatch):
    """What captured calls make is held for their graph's sake until vox_graph_destroy, by a capture whose stream the call is on; what an eager call makes is not."""
    import gc
    import weakref
    destroyed = []
    monkeypatch.setattr(N, "_graph_memory", {})
    monkeypatch.setattr(N, "_parted", [])
    monkeypatch.setattr(N, "_capturing", {})

    class Capture:
        def __init__(self, records):
            self.held, self.records = [], lambda: records

    t = torch.zeros(8)
    assert N.hold(t) is t                                    # no capture
    for records in (False, True):
        N._capturing[t.device.index] = cap = Capture(records)
        assert N.hold(t) is t and len(cap.held) == records
        del N._capturing[t.device.index]
    refs = [weakref.ref(cap.held[0])]
    N._graph_memory[77] = cap.held
    del t, cap
    gc.collect()
    assert refs[0]() is not None
    N._destroy(destroyed.append, 5)                          # another graph: nothing of ours
    assert refs[0]() is not None
    handle = N.c_void_p(77)
    N._capturing[None] = Capture(True)                       # inside a capture: the memory waits for its end
    N._destroy(destroyed.append, handle)
    assert destroyed == [5, handle] and not N._graph_memory and len(N._parted) == 1 and refs[0]() is not None
    N._let_go(N._parted.pop())
    gc.collect()
    assert refs[0]() is None
    assert not hasattr(B, "_kept")


def test_plans_count_their_requests_when_asked():
    """A plan for dense attention does no work for the operators beside it."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from vox_serve_amd.flashinfer_utils import FlashInferDecodeWrapper, FlashInferPrefillWrapper
    ops = []

    class Count(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            ops.append(func.overloadpacket.__name__)
            return func(*args, **(kwargs or {}))

    w = FlashInferPrefillWrapper(None, 4, 2, 256, 16, device="cpu")
    with Count():
        w.plan(torch.tensor([0, 5, 5, 6]), torch.tensor([0, 1, 2, 4]), torch.arange(4).int(), torch.tensor([5, 6, 7]))
    assert "gt" not in ops and ops.count("sum") == 1          # (the rows' number)
    assert w._n_own() == 2 and w._n_own() == 2
    w.plan(torch.tensor([0, 1, 2]), torch.tensor([0, 1, 2]), torch.arange(2).int(), torch.tensor([1, 1]))
    assert w._n_own() == 2
    d = FlashInferDecodeWrapper(None, 4, 2, 256, 16, device="cpu")
    d.plan(torch.tensor([0, 1, 2, 4]), torch.arange(4).int(), torch.tensor([5, 6, 7]))
    assert d._n_own() == 3


def test_rope_table():
    """The angles that a caller hands to set_kv_cache_rope: those of apply_rope_pos_ids, for as many positions as are asked for."""
    from vox_serve_amd import flashinfer_utils as F
    t = F.rope_table(20000, 64, rope_theta=1e6, device="cpu")
    assert t.shape == (20000, 32, 2) and t.dtype is torch.float32 and t.is_contiguous()
    assert torch.equal(t[:8192], F._rope_table(torch.device("cpu"), 8192, 64, 1e6, 1.0, None))
    angle = torch.arange(20000, dtype=torch.float32)[:, None] * (1e6 ** (-torch.arange(32, dtype=torch.float64) / 32)).float()
    assert (t - torch.stack([angle.double().cos(), angle.double().sin()], -1)).abs().max() < 20000 * 2.0 ** -22     # (a step of a frequency, and of its product)
    far = F.rope_table(64, 128, rope_scale=8.0, rope_theta=5e5, device="cpu", low_freq_factor=1.0, high_freq_factor=4.0, old_context_len=8192)
    assert torch.equal(far, F._rope_table(torch.device("cpu"), 64, 128, 5e5, 8.0, (1.0, 4.0, 8192)))
    for bad in ((0, 64), (10, 63), (10, 0)):
        with pytest.raises(ValueError, match="rope_table"):
            F.rope_table(*bad, device="cpu")
    with pytest.raises(TypeError, match="unexpected"):
        F.rope_table(10, 64, device="cpu", theta=1.0)


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scales_whose_exponents_overflow_are_refused(scale):
    """Scores are taken in powers of two: a scale that is not finite times log2 e would make every weight NaN."""
    assert call("vox_block_attention", B._ATTEND, ATTEND, scale=scale) == 1
    assert b"scale" in N.lib().vox_last_error()


def test_sizes_beyond_a_launch_are_refused():
    """Rows whose number comes near 2^31, heads whose channels do: refused, not wrapped around on the way to a launch."""
    most = 2 ** 31 - 1
    wide = dict(kv_heads=65535, heads=65535, n_pages=1, n_rows=most, head_dim=64)
    for own in (0, 1):
        assert call("vox_block_select", B._SELECT, SELECT, **dict(wide, n_own=own)) == 1
        assert b"more than a launch" in N.lib().vox_last_error()
        assert call("vox_block_attention", B._ATTEND, ATTEND, **dict(wide, n_own=own)) == 1
        assert b"more than a launch" in N.lib().vox_last_error()
    assert call("vox_rope_append", B._APPEND, APPEND, heads=most) == 1
    assert call("vox_rope_append", B._APPEND, APPEND, heads=most, bounds=0) == 1
    assert call("vox_rope_append", B._APPEND, APPEND, heads=2 ** 24, head_dim=512, bounds=0, rot=0) == 1
    assert b"heads" in N.lib().vox_last_error()


def test_wrappers_refuse_bounds_of_other_pages():
    from vox_serve_amd.flashinfer_utils import FlashInferDecodeWrapper
    w = FlashInferDecodeWrapper(None, 4, 2, 256, 128, device="cpu")
    w.plan(torch.tensor([0, 1]), torch.arange(1).int(), torch.tensor([5]))
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for shape in ((1, 2, 3, 2, 64), (1, 2, 0, 2, 64), (1, 2, 256, 2, 64), (1, 2, 2, 64)):
        with pytest.raises(ValueError, match="pages of 128 tokens"):
            w.select_blocks(q, torch.zeros(shape, dtype=torch.int8), torch.zeros(shape[:3]), top=4)
