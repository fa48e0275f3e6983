"""Packed tokens and caches in pages: what the entries refuse before any device use, and the pages' bookkeeping."""
import ctypes as C

import numpy as np
import pytest

import rustorch_amd as ra
from rustorch_amd import _lib as L

P = 0x10000
FAR = 1 << 40  # an address apart from every other


def append(q=P, q_out=FAR, k_in=2 * FAR, k_out=None, v_in=3 * FAR, kp=4 * FAR, vp=5 * FAR, table=P, starts=None, positions=P, pos=0, axes=None, sections=None,
           n_axes=None, cos=P, sin=P, table_rows=64, tokens=4, batch=2, heads=4, n_kv=2, dim=64, n_pages=8, page=16, table_pages=4):
    err = L.RtErr()
    arr = None if sections is None else np.asarray(sections, dtype=np.int32)
    rc = L.lib().rt_qk_norm_rope_kv_append_paged_bf16(
        None, q, q_out, k_in, k_out, v_in, kp, vp, table, starts, positions, pos, axes, None if arr is None else arr.ctypes.data,
        (0 if arr is None else arr.size) if n_axes is None else n_axes, None, None, 1e-6, cos, sin, table_rows, tokens, batch, heads, n_kv, dim, n_pages, page,
        table_pages, C.byref(err))
    return rc, err


def decode(q=P, kp=4 * FAR, vp=5 * FAR, out=FAR, table=P, lens=P, shared_lens=None, shared=0, batch=2, heads=4, n_kv=2, dim=64, n_pages=8, page=16, table_pages=4,
           ws=6 * FAR, ws_bytes=1 << 40):
    err = L.RtErr()
    rc = L.lib().rt_gqa_decode_paged_bf16(None, q, kp, vp, out, table, lens, shared_lens, shared, batch, heads, n_kv, dim, n_pages, page, table_pages, ws, ws_bytes,
                                          C.byref(err))
    return rc, err


def prompt(batch=2, heads=4, tokens=8, dim=64, n_kv=2, q=P, k=2 * FAR, v=3 * FAR, starts=P, out=FAR):
    err = L.RtErr()
    s = ra.AttentionShape.new(batch, heads, tokens, dim)._c()
    return L.lib().rt_flash_forward_packed_bf16_dev(None, C.byref(s), n_kv, q, k, v, starts, out, C.byref(err)), err


@pytest.mark.parametrize("more", [dict(tokens=-1), dict(batch=-1), dict(heads=-4), dict(n_kv=-1), dict(dim=-64), dict(n_pages=-1), dict(table_pages=-1), dict(table_rows=-1),
                                  dict(n_axes=-1), dict(dim=8), dict(dim=72), dict(dim=272), dict(page=8), dict(page=24), dict(page=2048), dict(page=0), dict(page=-16),
                                  dict(sections=[8, 8, 8, 4, 4], axes=P), dict(sections=[40, -8], axes=P), dict(q=P + 2), dict(v_in=3 * FAR + 8), dict(kp=4 * FAR + 2),
                                  dict(q_out=P + 16), dict(k_out=2 * FAR + 16), dict(k_out=FAR), dict(kp=5 * FAR + 16), dict(vp=3 * FAR), dict(kp=P), dict(heads=65536),
                                  dict(q_out=2 * FAR), dict(table_pages=1 << 27)])
def test_append_refuses(more):
    assert append(**more)[0] == L.RT_ERR_UNSUPPORTED


def test_append_refuses_more_tokens_than_a_grid_has():
    rc, err = append(tokens=(1 << 25) + 2, batch=2)
    assert rc == L.RT_ERR_UNSUPPORTED and b"launch grid" in err.message


def test_append_refuses_with_the_reference_errors():
    assert append(dim=0)[0] == L.RT_ERR_ZERO_DIM
    for more in (dict(q=None), dict(q_out=None), dict(k_in=None), dict(v_in=None), dict(kp=None), dict(vp=None), dict(table=None), dict(cos=None), dict(sin=None),
                 dict(sections=[32], axes=None), dict(n_axes=2, axes=P)):
        assert append(**more)[0] == L.RT_ERR_NULL_POINTER, more
    for sections in ([16, 8], [32, 1], [0]):
        rc, err = append(sections=sections, axes=P)
        assert rc == L.RT_ERR_ROPE_WRONG_INPUT_LEN and (err.expected, err.got) == (32, sum(sections))
    rc, err = append(tokens=5)
    assert rc == L.RT_ERR_WRONG_INPUT_LEN and (err.expected, err.got) == (2, 5)
    rc, err = append(positions=None, pos=63)
    assert rc == L.RT_ERR_ROPE_POSITION_OVERFLOW and (err.expected, err.got) == (64, 65)
    assert append(positions=None, pos=-1)[0] == L.RT_ERR_ROPE_POSITION_OVERFLOW
    rc, err = append(positions=None, pos=63, table_rows=100)
    assert rc == L.RT_ERR_KV_OVERFLOW and (err.expected, err.got) == (64, 65)
    assert append(positions=None, pos=63, sections=[32], axes=P)[0] == L.RT_ERR_KV_OVERFLOW  # the tables are not asked there
    assert append(positions=None, pos=65, starts=P, table_rows=100)[0] == L.RT_ERR_KV_OVERFLOW


def test_append_checks_the_lowest_row_of_packed_sequences():
    """A host position with `starts`: the row of the first token there may be, ahead of the tables' and the page table's last."""
    for more, status in ((dict(pos=64), L.RT_ERR_ROPE_POSITION_OVERFLOW), (dict(pos=64, table_rows=65), L.RT_ERR_KV_OVERFLOW), (dict(pos=64, sections=[32], axes=P), L.RT_ERR_KV_OVERFLOW)):
        rc, err = append(positions=None, starts=P, **more)
        assert rc == status and (err.expected, err.got) == (64, 65), more
    assert append(positions=None, starts=P, pos=64, tokens=0)[0] == L.RT_OK


def test_append_of_nothing_is_done():
    assert append(tokens=0)[0] == L.RT_OK and append(batch=0, tokens=7)[0] == L.RT_OK and append(heads=0, n_kv=0)[0] == L.RT_OK


def test_calls_that_are_right_get_as_far_as_the_device():
    done = (L.RT_ERR_NO_DEVICE,)
    if L.lib().rt_init(0, C.byref(L.RtErr())) == 0:
        pytest.skip("the addresses are no memory")
    for more in (dict(), dict(q_out=P), dict(k_out=2 * FAR), dict(starts=P, tokens=5), dict(sections=[16, 8, 8], axes=P), dict(sections=[0, 32], axes=P), dict(dim=256), dict(page=1024)):
        assert append(**more)[0] in done, more
    for more in (dict(), dict(shared=64), dict(shared_lens=P, shared=-1), dict(heads=40, n_kv=1), dict(dim=16)):
        assert decode(**more)[0] in done, more
    assert prompt()[0] in done and prompt(n_kv=0)[0] in done and prompt(dim=8)[0] in done


@pytest.mark.parametrize("more", [dict(batch=-1), dict(heads=-4), dict(n_kv=-2, heads=-4), dict(dim=-1), dict(n_pages=-1), dict(table_pages=-1), dict(dim=8), dict(dim=72), dict(dim=264),
                                  dict(page=15), dict(page=8), dict(page=4096), dict(batch=65536), dict(table_pages=1 << 25), dict(batch=65535, table_pages=1 << 16),
                                  dict(q=P + 8), dict(out=FAR + 2), dict(kp=4 * FAR + 2), dict(vp=5 * FAR + 4)])
def test_decode_refuses(more):
    assert decode(**more)[0] == L.RT_ERR_UNSUPPORTED


@pytest.mark.parametrize("more", [dict(out=P), dict(out=4 * FAR + 64), dict(out=5 * FAR), dict(out=6 * FAR + 256), dict(ws=P), dict(ws=4 * FAR - 256), dict(ws=5 * FAR + 1024)])
def test_decode_refuses_outputs_over_inputs(more):
    rc, err = decode(**more)
    assert rc == L.RT_ERR_UNSUPPORTED and b"share no memory" in err.message


@pytest.mark.parametrize("more", [dict(table=FAR), dict(table=FAR - 28), dict(lens=FAR + 4), dict(lens=FAR - 4), dict(lens=6 * FAR + 16), dict(table=6 * FAR + 64), dict(shared_lens=FAR + 8),
                                  dict(shared_lens=6 * FAR)])
def test_decode_refuses_outputs_over_its_table_and_lengths(more):
    """What every workgroup reads, the second launch too: none may write there.  (Table of 2 x 4 entries, two lengths, one prefix.)"""
    rc, err = decode(**more)
    assert rc == L.RT_ERR_UNSUPPORTED and b"share no memory" in err.message


def test_packed_prompts_refuse_an_output_over_their_starts():
    for starts in (FAR, FAR + 64, FAR - 8):  # three of them
        rc, err = prompt(starts=starts)
        assert rc == L.RT_ERR_UNSUPPORTED and b"share no memory" in err.message


def test_decode_refuses_with_the_reference_errors():
    assert decode(dim=0)[0] == L.RT_ERR_ZERO_DIM
    assert decode(heads=4, n_kv=3)[0] == decode(n_kv=0)[0] == L.RT_ERR_HEAD_COUNT_MISMATCH
    for more in (dict(q=None), dict(out=None), dict(lens=None), dict(table=None), dict(kp=None), dict(vp=None)):
        assert decode(**more)[0] == L.RT_ERR_NULL_POINTER, more
    for shared in (-1, 65):
        rc, err = decode(shared=shared)
        assert rc == L.RT_ERR_KV_OVERFLOW and err.expected == 64
    need = ra.LlmKernels.gqa_decode_paged_workspace_bytes(2, 4, 2, 64, 16, 4)
    assert need > 0
    rc, err = decode(ws_bytes=need - 1)
    assert rc == L.RT_ERR_WORKSPACE_TOO_SMALL and (err.expected, err.got) == (need, need - 1)
    assert decode(ws=None)[0] == decode(ws=6 * FAR + 8)[0] == L.RT_ERR_WORKSPACE_TOO_SMALL
    assert decode(batch=0)[0] == decode(heads=0)[0] == L.RT_OK
    for bad in ((0, 4, 2, 64, 16, 4), (2, 4, 3, 64, 16, 4), (2, 4, 2, 72, 16, 4), (2, 4, 2, 64, 20, 4), (2, 4, 2, 64, 16, -1)):
        assert ra.LlmKernels.gqa_decode_paged_workspace_bytes(*bad) == 0


def test_packed_prompts_refuse():
    assert prompt(dim=0)[0] == L.RT_ERR_ZERO_DIM
    assert prompt(n_kv=3)[0] == L.RT_ERR_HEAD_COUNT_MISMATCH
    for more in (dict(dim=12), dict(dim=264), dict(q=P + 2), dict(k=2 * FAR + 8), dict(out=FAR + 4), dict(batch=65536), dict(tokens=1 << 32), dict(tokens=1 << 24, dim=128),
                 dict(out=P), dict(out=2 * FAR), dict(out=3 * FAR + 16)):
        assert prompt(**more)[0] == L.RT_ERR_UNSUPPORTED, more
    for name in ("q", "k", "v", "starts", "out"):
        assert prompt(**{name: None})[0] == L.RT_ERR_NULL_POINTER
    assert prompt(batch=0)[0] == prompt(heads=0)[0] == prompt(tokens=0)[0] == L.RT_OK


class NoPages(ra.PagedKVCache):
    """The bookkeeping alone: no layers, no device."""

    def __init__(self, max_sequences, n_pages, page_size=16, table_pages=None):
        super().__init__(0, max_sequences, 2, 64, n_pages, page_size, table_pages)


def test_pages_are_given_shared_and_taken_back():
    c = NoPages(3, 8)
    a = c.add()
    c.reserve(a, 33)
    c.advance(a, 33)
    assert c.free_pages() == 5 and c.length(a) == 33
    b = c.add(prefix_of=a, shared=32)
    assert c.length(b) == 32 and c.free_pages() == 5
    c.reserve(b, 1)
    t = c.table([a, b])
    assert (t[0, :2] == t[1, :2]).all() and t[0, 2] != t[1, 2] and (t[:, 3:] == -1).all()
    assert c.table([b], write_from=[32])[0, :3].tolist() == [-1, -1, t[1, 2]] and c.table([a], write_from=[31])[0, 1] == t[0, 1]
    c.remove(a)
    assert c.free_pages() == 5  # b has the others
    c.remove(b)
    assert c.free_pages() == 8
    with pytest.raises(KeyError):
        c.length(a)


def test_pages_run_out():
    c = NoPages(2, 4, table_pages=3)
    a = c.add()
    with pytest.raises(ra.Overflow):
        c.reserve(a, 49)  # the table's row
    c.reserve(a, 48)
    b = c.add()
    with pytest.raises(ra.Overflow):
        c.add()
    with pytest.raises(ra.Overflow):
        c.reserve(b, 17)
    assert c.free_pages() == 1  # none was taken
    c.reserve(b, 16)
    with pytest.raises(ra.Overflow):
        c.advance(b, 17)
    with pytest.raises(ra.Overflow):
        c.advance(b, -1)
    with pytest.raises(ValueError):
        c.reserve(b, -1)
    c.remove(b)
    for shared in (16, 1, -16):
        with pytest.raises((ra.Overflow, ValueError)):
            c.add(prefix_of=a, shared=shared)  # a has no rows yet; not a whole page
    with pytest.raises(ra.LayerOutOfRange):
        c.layer(0)
    with pytest.raises(KeyError):
        c.add(prefix_of=1, shared=16)


class Calls:
    """What reaches the append's native entry."""

    def __init__(self, monkeypatch):
        self.seen = []
        monkeypatch.setattr(L, "native", self)

    def rt_qk_norm_rope_kv_append_paged_bf16(self, *args):
        at, n = args[13], args[14]
        self.seen.append(None if at is None else list((C.c_int32 * n).from_address(at)))


class Rope:
    max_seq = 64

    def device_tables(self):
        return P, P


def append_call(sections, rope=None, dim=64):
    ra.LlmKernels.qk_norm_rope_kv_append_paged_bf16(None, P, FAR, 2 * FAR, 3 * FAR, ra.KVPages(4 * FAR, 5 * FAR, 8, 16), P, 4, P, rope or Rope(), 4, 2, 4, 2, dim,
                                                    axis_positions=None if sections is None else P, sections=sections)


def test_sections_are_the_numbers_that_a_call_is_given(monkeypatch):
    """Whatever holds them, and whatever it held in the call before."""
    calls = Calls(monkeypatch)
    held = np.array([[8], [24]], dtype=np.int64)
    for first in (8, 10):
        held[:, 0] = first, 32 - first
        append_call(held[:, 0])
        append_call([int(x) for x in held[:, 0]])
    assert calls.seen == [[8, 24], [8, 24], [10, 22], [10, 22]]

    class Number:  # an integer by its protocol, as a tensor of one element is
        def __init__(self, value):
            self.value = value

        def __index__(self):
            return self.value

        def __int__(self):
            return self.value

    calls.seen.clear()
    mine = [Number(8), Number(24)]
    append_call(mine)
    mine[0].value, mine[1].value = 16, 16
    append_call(mine)
    assert calls.seen == [[8, 24], [16, 16]]
    calls.seen.clear()
    append_call([8.0, np.float64(24)])
    append_call(held[:, 0].tolist() + [np.int32(0)])
    append_call(x for x in (Number(8), 24))
    assert calls.seen == [[8, 24], [10, 22, 0], [8, 24]]
    for bad in ([16.5, 15.5], ["8", "24"], [float("nan"), 32]):
        with pytest.raises(TypeError):
            append_call(bad)


def test_tables_of_another_head_dim_are_refused(monkeypatch):
    """The kernel takes half a head's angles a row: rows of fewer would be read past the tables' end, of more give others' angles."""
    calls = Calls(monkeypatch)

    class Of32(Rope):
        head_dim = 32

    for dim in (64, 16):
        with pytest.raises(ra.RopeWrongInputLen) as e:
            append_call(None, Of32(), dim)
        assert (e.value.expected, e.value.got) == (64 * dim // 2, 64 * 16)
    with pytest.raises(ra.RopeWrongInputLen):
        append_call(None, ra.RoPE(128, 64), 64)
    assert not calls.seen
    append_call(None, Of32(), 32)
    append_call(None)  # (tables that do not say what they are of)
    assert calls.seen == [None, None]


def test_write_from_is_a_row_for_each_sequence():
    """Fewer left the rest of the table's rows writable, a row below 0 cut the table from its end."""
    c = NoPages(3, 8)
    a = c.add()
    c.reserve(a, 48)
    c.advance(a, 40)
    b = c.add(prefix_of=a, shared=32)
    c.reserve(b, 1)
    for bad in ([32], [], [40, 32, 0], [-1, 32], [40, -17]):
        with pytest.raises(ValueError):
            c.table([a, b], write_from=bad)
    t = c.table([a, b])
    got = c.table([a, b], write_from=np.array([0, 32], dtype=np.int32))
    assert (got[0] == t[0]).all() and got[1].tolist()[:3] == [-1, -1, t[1, 2]]
    assert (c.table([b, a], write_from=c.lengths([b, a]))[:, :2] == -1).all()  # a row past what it has: nothing ahead of it
    assert c.table([], write_from=[]).shape == (0, 8)
    assert (c.table(iter([a, b]), write_from=iter([0, 32])) == got).all() and c.lengths(iter([a, b])).tolist() == [40, 32]
