"""The paged 4-bit cache without a GPU: its layout, where a position lies, what the library and the wrappers
refuse, the books that `PagedCache` keeps."""
import ctypes as C

import pytest
import torch

import paged_plain as P
from shard_b200 import _lib, ops
from shard_b200._lib import ShardError, ShardPaged


def _cache(table, n_pages=10, nkv=3, page_size=32, **over):
    """A ShardPaged over host memory that no call here reads but the table."""
    table = torch.as_tensor(table, dtype=torch.int32)
    c = ShardPaged(4096, table.data_ptr(), 4096, 4096, table.stride(0), table.shape[1], table.shape[0], n_pages, page_size, nkv, 0)
    for name, value in over.items():
        setattr(c, name, value)
    return c, table


def test_every_byte_of_a_block_has_one_meaning():
    codes = P.code_at()
    places = torch.cat([(codes * 2 + torch.arange(128) % 2).flatten() + 2048 * v for v in (0, 1)])
    assert torch.equal(places.sort().values, torch.arange(4096))
    words = torch.cat([P.param_at(v).flatten() for v in (False, True)])
    assert torch.equal(words.sort().values, torch.arange(2048, 2176, 2))
    assert C.sizeof(ShardPaged) == 4 * 8 + 8 + 6 * 4


def test_four_bits_times_seven_are_an_fp16_number():
    """Every value that a code can stand for is exact in fp16, whatever the scale."""
    s = (torch.arange(0, 0x7c00, 16, dtype=torch.int16).view(torch.float16)).double()
    s = s[s * 15 < 65504]
    v = s[:, None] * torch.arange(-15, 16)
    assert torch.equal(v.half().double(), v)


@pytest.mark.parametrize("spread", [1.0, 30.0, 1e-3, 5e-7, 3e4, 1e9])
def test_error_of_the_quantisation(spread):
    """Half a step from rounding; the scale's own rounding (2^-7 of it and fp16's 2^-11, 15 steps long) moves the
    ends by an eighth of a step more, where the codes stop; below fp16's normal range scales are multiples of 2^-20."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(400, 128, generator=g) * spread
    x[:40] = x[:40].abs()
    x[40:60, 17] *= 100
    code, s, z = P.quantise(x)
    x = x.clamp(-32768, 32768).view(400, 2, 64).double()
    err = (P.held(x.flatten(1).float()).view(400, 2, 64) - x).abs().amax(-1)
    step = torch.where(s > 0, s, 0.0).double()
    assert (err <= 0.5 * step + 15 * (step * (2.0 ** -7 + 2.0 ** -10)) + 15 * 2.0 ** -21).all()
    assert code.min() >= 0 and code.max() <= 15 and z.max() <= 15


def test_where_a_position_lies():
    lib = _lib.load()
    table = [[3, 0, 9, -1], [10, 2 ** 31 - 1, -2 ** 31, 5]]
    c, keep = _cache(table)
    at = lambda seq, pos, head: lib.shard_b200_paged_offset(C.byref(c), seq, pos, head)
    page = lib.shard_b200_paged_page_bytes(3, 32)
    assert page == 3 * 2 * 2176
    for seq in (0, 1):
        for pos in (0, 1, 15, 16, 31, 32, 63, 64, 95, 96, 127):
            entry = table[seq][pos // 32]
            for head in (0, 2):
                want = entry * page + (head * 2 + pos % 32 // 16) * 2176 if 0 <= entry < 10 else -1
                assert at(seq, pos, head) == want, (seq, pos, head)
    for seq, pos, head in ((0, -1, 0), (0, 128, 0), (0, 2 ** 31 - 1, 0), (0, -2 ** 31, 0), (-1, 0, 0), (2, 0, 0), (0, 0, 3), (0, 0, -1)):
        assert at(seq, pos, head) == -1
    # a pool of more than 4 GiB
    c, keep = _cache([[400000]], n_pages=400001, nkv=8, page_size=128)
    assert at(0, 127, 7) == 400000 * 8 * 8 * 2176 + 7 * 8 * 2176 + 7 * 2176
    # rows of the table that are apart
    wide = torch.arange(12, dtype=torch.int32).view(2, 6)
    c, keep = _cache(wide[:, :4])
    assert c.table_stride == 6 and at(1, 0, 0) == 6 * page


def test_library_refuses():
    lib = _lib.load()
    good, keep = _cache([[0]])
    assert lib.shard_b200_paged_page_bytes(0, 64) == 0 and lib.shard_b200_paged_page_bytes(2, 48) == 0
    assert lib.shard_b200_paged_page_bytes(2, 256) == 0 and lib.shard_b200_paged_page_bytes(2, 8) == 0
    buf = 4096

    def append(c=good, k=buf, v=buf, q=None, strides=(128,) * 6, n_q=0, rows=1, dtype=0, rope=buf, rope_rows=8, q_out=None):
        return lib.shard_b200_paged_append(C.byref(c) if c else None, k, v, q, *strides, n_q, rows, dtype, rope, rope_rows, q_out, None, None)

    def attn(c=good, q=buf, strides=(128, 128), n_q=6, rows=1, max_new=1, dtype=0, scale=0.1, out=buf, lse=None, ws=buf, wsb=1 << 40):
        return lib.shard_b200_paged_attn(C.byref(c) if c else None, q, *strides, n_q, rows, max_new, dtype, scale, out, lse, ws, wsb, None, None)

    def read(c=good, rows=1, dtype=0, k=buf, v=buf):
        return lib.shard_b200_paged_read_back(C.byref(c) if c else None, rows, dtype, k, v, None, None)

    bad = [dict(pool=None), dict(page_table=None), dict(cu=None), dict(lens=None), dict(n_seqs=-1), dict(n_seqs=8193), dict(nkv=0),
           dict(page_size=48), dict(page_size=0), dict(n_pages=-1), dict(table_width=2), dict(table_width=-1)]
    for over in bad:
        c, keep2 = _cache([[0]], **over)
        assert append(c) == attn(c) == read(c) == -1, over
        assert lib.shard_b200_paged_attn_workspace_bytes(C.byref(c), 6, 1, 1) == 0
    c, keep2 = _cache([[0]], pool=4104)
    assert append(c) == attn(c) == read(c) == -3
    assert append(None) == attn(None) == read(None) == -1
    assert append(k=None) == append(v=None) == append(rope=None) == append(rows=-1) == append(dtype=2) == append(rope_rows=-1) == -1
    assert append(q=buf, n_q=6) == append(q=buf, q_out=buf, n_q=0) == -1
    assert append(k=4100) == append(rope=4100) == append(strides=(128, 132, 128, 128, 0, 0)) == -3
    assert append(q=buf, q_out=buf, n_q=6, strides=(128, 128, 128, 128, 4, 8)) == -3
    assert attn(q=None) == attn(out=None) == attn(ws=None) == attn(n_q=0) == attn(n_q=7) == attn(max_new=-1) == attn(dtype=7) == -1
    assert attn(scale=float("nan")) == attn(scale=float("inf")) == -1
    assert attn(wsb=0) == -2
    assert attn(q=4100) == attn(out=4100) == attn(ws=4100) == attn(lse=4098) == attn(strides=(4, 128)) == -3
    assert read(k=None) == read(v=None) == read(dtype=-1) == -1 and read(k=4112) == -3
    # calls without work
    assert append(rows=0) == attn(rows=0) == read(rows=0) == 0
    c, keep2 = _cache([[0]], n_seqs=0)
    assert append(c) == attn(c) == read(c) == 0


def test_wrappers_refuse_cpu_tensors():
    pool = torch.zeros(2, 1, 2176, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ShardError):
        ops.paged_read_back(pool, i[:1].view(1, 1), i, i[:1], 1)


@pytest.fixture
def on_cpu(monkeypatch):
    """The wrappers' checks with tensors of the CPU in the place of the GPU's; no kernel is launched."""
    monkeypatch.setattr(ops, "require_cuda", lambda *t: None)
    launched = []
    class Lib:
        def __getattr__(self, name):
            def call(*a):
                launched.append(name)
                return 64 if name.endswith("bytes") else 0
            return call
    monkeypatch.setattr(ops._lib, "load", lambda: Lib())
    monkeypatch.setattr(ops, "cur_stream", lambda: 0)
    return launched


def test_wrappers_refuse(on_cpu):
    pool, table = torch.zeros(4, 2, 4352, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.int32)
    cu, lens = torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    kv, q = torch.zeros(5, 2, 128, dtype=torch.float16), torch.zeros(5, 6, 128, dtype=torch.float16)
    rope = torch.zeros(9, 128)
    meta = (pool, table, cu, lens)
    ops.paged_append(kv, kv, *meta, rope, q=q)
    ops.paged_attn(q, *meta)
    ops.paged_read_back(*meta, 5)
    assert [n for n in on_cpu if not n.endswith("bytes")] == ["shard_b200_paged_append", "shard_b200_paged_attn", "shard_b200_paged_read_back"]
    for m in ((pool.int(), table, cu, lens), (pool[:, :, :100], table, cu, lens), (pool.transpose(0, 1), table, cu, lens),
              (pool.new_zeros(4, 2, 3 * 2176), table, cu, lens), (pool, table.long(), cu, lens), (pool, table[:2], cu, lens),
              (pool, table.t().contiguous().t(), cu, lens), (pool, table, cu[:3], lens), (pool, table, cu, lens.float()),
              (pool, table, cu.new_zeros(8)[::2], lens), (pool, table[:1].expand(3, 2), cu, lens),
              (pool, table.new_zeros(8193, 1), cu.new_zeros(8194), lens.new_zeros(8193)), (pool[:0], table, cu, lens),
              (pool, table.new_zeros(1, 1).expand(3, 1 << 26), cu, lens)):
        with pytest.raises(ShardError):
            ops.paged_read_back(*m, 5)
    for a, kw in (((kv.float(), kv.float(), *meta, rope), {}), ((kv, kv.bfloat16(), *meta, rope), {}), ((kv, kv[:4], *meta, rope), {}),
                  ((kv[:, :1], kv, *meta, rope), {}), ((kv[..., :64], kv, *meta, rope), {}), ((kv, kv, *meta, rope.double()), {}),
                  ((kv, kv, *meta, rope[:, :64]), {}), ((kv, kv, *meta, rope.t().contiguous().t()), {}),
                  ((kv, kv, *meta, rope), dict(q=q[:4])), ((kv, kv, *meta, rope), dict(q=q.bfloat16())),
                  ((kv, kv, *meta, rope), dict(q=q, q_out=q[:, :3])), ((kv, kv, *meta, rope), dict(status=rope))):
        with pytest.raises(ShardError):
            ops.paged_append(*a, **kw)
    for a, kw in (((q[:, :5], *meta), {}), ((q[:, :0], *meta), {}), ((q.float(), *meta), {}), ((q, *meta), dict(out=q.bfloat16())),
                  ((q, *meta), dict(out=torch.zeros(5, 128, 6, dtype=torch.float16).transpose(1, 2))),
                  ((q, *meta), dict(lse=torch.zeros(5, 5))), ((q, *meta), dict(max_new=-1))):
        with pytest.raises(ShardError):
            ops.paged_attn(*a, **kw)
    with pytest.raises(ShardError):
        ops.paged_read_back(*meta, 5, dtype=torch.float32)
    # calls without work launch nothing
    on_cpu.clear()
    none = (pool, table[:0], cu[:1], lens[:0])
    assert ops.paged_attn(q[:0], *meta).shape == (0, 6, 128) and ops.paged_append(kv[:0], kv[:0], *meta, rope) is None
    assert ops.paged_attn(q, *none).shape == q.shape and ops.paged_read_back(*none, 5)[0].shape == (5, 2, 128)
    assert not [n for n in on_cpu if not n.endswith("bytes")]


def test_views_that_the_kernels_cannot_read_are_copied(on_cpu):
    odd = torch.zeros(5 * 2 * 128 + 1, dtype=torch.float16)[1:].view(5, 2, 128)
    assert ops._paged_rows(odd, 2, None, "keys").data_ptr() % 16 == 0
    apart = torch.zeros(5, 2, 129, dtype=torch.bfloat16)[..., :128]
    assert ops._paged_rows(apart, 2, None, "keys").is_contiguous()
    cut = torch.zeros(5, 10, 128, dtype=torch.float16)[:, 6:8]
    assert ops._paged_rows(cut, 2, None, "keys") is cut


def test_books_of_the_pages():
    from shard_b200 import PagedCache
    c = PagedCache(2, 2, 10, 3, 100, torch.ones(64), page_size=16, device="cpu")
    assert c.pools.shape == (2, 10, 2, 2176) and c.rope.shape == (100, 128)
    a, b = c.add(), c.add()
    c.begin({a: 17, b: 3})
    table, cu, lens, rows, most = c._batch
    assert rows == 20 and most == 17 and cu.tolist() == [0, 17, 20] and lens.tolist() == [17, 3] and table.shape == (2, 2)
    assert c.free_pages == 7 and table[1, 1] == -1 and len({*table.flatten().tolist()} - {-1}) == 3
    with pytest.raises(ShardError):
        c.begin({a: 84})                       # more than max_len
    with pytest.raises(ShardError):
        c.begin({a: 80, b: 60})                # 5 + 3 pages of the 7 that are free
    with pytest.raises(ShardError):
        c.begin({a: 1, 2: 1})                  # no such sequence
    with pytest.raises(ShardError):
        c.begin({a: -1})
    assert c.length(a) == 17 and c.length(b) == 3 and c.free_pages == 7
    with pytest.raises(ShardError):
        c.append(0, torch.zeros(19, 2, 128), torch.zeros(19, 2, 128))
    c.begin({b: 13, a: 0})
    assert c._batch[1].tolist() == [0, 13, 13] and c.length(b) == 16 and c.free_pages == 7
    assert c.memory_bytes() == 3 * 2 * 2 * 2176 and c.fp16_equivalent_bytes() == 33 * 2 * 2 * 512
    held = set(c._slots[a])
    c.remove(a)
    assert c.free_pages == 9 and held <= set(c._free)
    with pytest.raises(ShardError):
        c.append(0, torch.zeros(1, 2, 128), torch.zeros(1, 2, 128))      # begin() comes first
    with pytest.raises(ShardError):
        c.length(a)
    assert c.add() == a and c.length(a) == 0 and c.add() == 2
    with pytest.raises(ShardError):
        c.add()
    with pytest.raises(ShardError):
        PagedCache(1, 2, 10, 3, 100, device="cpu")
    with pytest.raises(ShardError):
        PagedCache(1, 2, 10, 3, 100, rope=torch.zeros(99, 128), device="cpu")
    with pytest.raises(ShardError):
        PagedCache(1, 2, 10, 3, 100, torch.ones(64), page_size=20, device="cpu")


def test_begin_refuses_too_many_sequences_and_captures(monkeypatch):
    from shard_b200 import PagedCache
    c = PagedCache(1, 1, 1, 8193, 16, torch.ones(64), page_size=16, device="cpu")
    with pytest.raises(ShardError):
        c.begin({c.add(): 0 for _ in range(8193)})
    c.begin({s: 0 for s in range(8192)})
    assert c._batch[0].shape == (8192, 0) and c._batch[3] == 0
    c.begin({})
    assert c._batch[0].shape[0] == 0 and c._batch[1].tolist() == [0]
    c.device = torch.device("cuda")            # (refused before anything is copied)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: c.begin({0: 1}), lambda: c.read_back(0, 0)):
        with pytest.raises(ShardError, match="capture"):
            call()
    assert c.length(0) == 0 and c.free_pages == 1


def test_rotation_table():
    from shard_b200.rope import reapply_rope, rope_table
    inv = 1.0 / (500000.0 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    x = torch.randn(7, 128, generator=torch.Generator().manual_seed(1))
    pos = torch.tensor([0, 1, 5, 77, 1000, 8190, 8191])
    t = rope_table(8192, inv)[pos]
    assert torch.equal(P.rotate(x[:, None], t[:, :64], t[:, 64:])[:, 0], reapply_rope(x, pos, inv))


def test_books_of_truncated_sequences():
    from shard_b200 import PagedCache
    c = PagedCache(1, 2, 6, 2, 100, torch.ones(64), page_size=16, device="cpu")
    a, b = c.add(), c.add()
    c.begin({a: 40, b: 16})
    first, freed = c._slots[a][:2], c._slots[a][2]
    for tokens in (41, -1):
        with pytest.raises(ShardError):
            c.truncate(a, tokens)
    assert c.length(a) == 40 and c.free_pages == 2 and c._batch is not None
    c.truncate(a, 33)                          # the third page still holds a token
    assert c.length(a) == 33 and c.free_pages == 2 and c._slots[a] == first + [freed]
    with pytest.raises(ShardError):
        c.append(0, torch.zeros(56, 2, 128), torch.zeros(56, 2, 128))      # begin() comes first
    c.truncate(a, 32)
    assert c.length(a) == 32 and c.free_pages == 3 and c._slots[a] == first
    c.begin({b: 1, a: 1})
    assert c._slots[b][1] == freed and c._batch[2].tolist() == [17, 33] and len({*c._slots[a], *c._slots[b]}) == 5
    c.truncate(b, 0)
    assert c.length(b) == 0 and c.free_pages == 3 and c._slots[b] == []
    c.begin({b: 20})
    assert c.length(b) == 20 and c.memory_bytes() == 5 * 2 * 2176
    c.remove(b)
    c.truncate(a, 33)
    assert c.length(a) == 33 and c.free_pages == 3
    with pytest.raises(ShardError):
        c.truncate(b, 0)
