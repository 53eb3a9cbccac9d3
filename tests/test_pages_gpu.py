"""The page operations (ada_pages_*) against a sequential model of their
documentation: tables, lengths, reference counts and page data, all equal."""

import pytest
import torch

import adaattn_b200 as ada
from adaattn_b200 import _lib
from serving_util import PoolModel

pytestmark = pytest.mark.gpu


class Pool:
    """A pool on the device and its model side by side."""

    def __init__(self, lens, page, *, slots, width, pages, dev, dtype=torch.bfloat16, block=(2, 5), planes=3, seed=0):
        g = torch.Generator().manual_seed(seed)
        ids = torch.randperm(pages, generator=g).tolist()
        table = torch.full((slots, width), -1, dtype=torch.int32)
        ln = torch.zeros(slots, dtype=torch.int32)
        refs = torch.zeros(pages, dtype=torch.int32)
        for s, n in enumerate(lens):
            ln[s] = n
            for j in range(-(-n // page)):
                p = ids.pop()
                table[s, j], refs[p] = p, 1
        data = torch.randn(planes, pages, block[0], page, block[1], generator=g).to(dtype)
        self.m = PoolModel(table, ln, refs, data, page)
        self.table, self.lens, self.refs, self.data = (t.to(dev) for t in (table, ln, refs, data))
        self.dev, self.page = dev, page

    def ids(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    @property
    def pool(self):
        return self.table, self.lens, self.refs

    def free(self, seqs):
        ada.free_pages(*self.pool, self.ids(seqs), page_size=self.page)
        self.m.free(seqs)

    def fork(self, src, dst):
        ada.fork_pages(*self.pool, self.ids(src), self.ids(dst), page_size=self.page)
        self.m.fork(src, dst)

    def copy(self, src, dst):
        got = ada.copy_pages(self.data, *self.pool, self.ids(src), self.ids(dst))
        assert got.tolist() == self.m.copy(src, dst)

    def reserve(self, seqs, new):
        got = ada.reserve_pages(self.data, *self.pool, self.ids(seqs), self.ids(new))
        want = self.m.reserve(seqs, new)
        assert got.tolist() == want
        return want

    def compact(self):
        got = ada.compact_pages(self.data, *self.pool)
        assert int(got) == self.m.compact()

    def check(self, clean=True):
        torch.cuda.synchronize()
        if clean:
            _lib.poll_device_status(self.dev)
        else:
            with pytest.raises(ada.KernelError):
                _lib.poll_device_status(self.dev)
        m = self.m
        assert torch.equal(self.lens.cpu(), m.lens)
        assert torch.equal(self.refs.cpu(), m.refs)
        assert torch.equal(self.table.cpu(), m.table)
        assert torch.equal(self.data.cpu().view(torch.uint8), m.data.view(torch.uint8))


@pytest.mark.parametrize("dtype,block,page", [(torch.bfloat16, (2, 64), 16), (torch.float32, (1, 3), 5),
                                              (torch.float8_e4m3fn, (3, 1), 3), (torch.float16, (1, 1), 1),
                                              (torch.float8_e4m3fn, (8, 128), 64)])
def test_fork_reserve_free(dtype, block, page, cuda_device):
    p = Pool([0, 1, page, page + 1, 3 * page - 1, 2 * page], page, slots=12, width=6, pages=60, dev=cuda_device,
             dtype=dtype, block=block, seed=page)
    p.fork([0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 11])
    p.check()
    p.reserve([6, 7, 8, 9, 10, 11], [1, 0, 2, page, 1, 2 * page])
    p.check()
    p.reserve([1, 3, 4], [1, 1, 1])   # sole holders again, except of the untouched fork
    p.check()
    p.free([0, 6, 3, 9])
    p.check()
    p.fork([4, 4, 4], [0, 3, 6])      # several branches of one sequence
    p.reserve([0, 3, 6, 4], [1, 1, 1, 1])   # all holders grow: the last keeps the page
    p.check()
    p.compact()
    p.check()
    p.copy([4, 11, 1], [2, 5, 8])
    p.check()


def test_reserve_runs_out_in_order(cuda_device):
    p = Pool([3, 0, 4, 2], 4, slots=6, width=8, pages=8, dev=cuda_device)
    # 3 pages held, 5 free; needs 2 + 2 fit, 3 does not, a need of none is still served
    assert p.reserve([0, 1, 2, 3], [8, 5, 12, 2]) == [8, 5, 0, 2]
    p.check()
    assert p.reserve([2], [4]) == [4]
    p.check()
    assert p.reserve([2, 3], [1, 1]) == [0, 0]
    p.check()
    p.free([0, 1, 2, 3])
    p.check()
    assert p.refs.sum().item() == 0


def test_the_last_holder_waits_for_the_copies(cuda_device):
    """Two holders of a part-full page, no page free: neither may write to it."""
    p = Pool([2], 4, slots=3, width=4, pages=1, dev=cuda_device)
    p.fork([0], [1])
    assert p.reserve([0, 1], [1, 1]) == [0, 0]
    p.check()
    p = Pool([2], 4, slots=3, width=4, pages=2, dev=cuda_device)
    p.fork([0], [1])
    assert p.reserve([1, 0], [1, 1]) == [1, 1]
    p.check()


def test_ids_named_twice_out_of_range_and_chains(cuda_device):
    p = Pool([5, 9, 2, 7], 4, slots=8, width=6, pages=40, dev=cuda_device)
    p.fork([0, 1, 2], [4, 4, 5])          # 4 twice: the first counts
    p.check(clean=False)
    p.fork([0, 6, 1], [6, 7, 1])          # 6 and 1 are also sources, 0 -> 6 and 1 -> 1 are left out
    p.check(clean=False)
    p.fork([-1, 9, 0, 0], [6, 6, 8, -3])  # out of range (and 6 is taken by the first pair that names it)
    p.check(clean=False)
    p.copy([0, 1, 3, 2], [6, 6, 7, 3])
    p.check(clean=False)
    p.reserve([0, 0, 9, 2], [1, 2, 1, 1])
    p.check(clean=False)
    p.reserve([0, 1], [-1, 1000])         # shrinking and more than the table holds
    p.check(clean=False)
    p.free([0, 0, 1])                     # freed once
    p.check()
    p.free([-1, 8, 2])
    p.check(clean=False)


def test_copy_runs_out_and_reuses_the_destinations(cuda_device):
    p = Pool([8, 12, 6], 4, slots=5, width=4, pages=13, dev=cuda_device)
    p.reserve([3], [16])                   # 3 + 2 + 2 + 4 = 11 pages held
    p.copy([0, 1, 2], [3, 4, 3])           # 3's four pages come back: 6 free for 2 + 3
    p.check(clean=False)
    p.free([3])
    p.copy([1, 0], [3, 4])
    p.check()
    p.copy([1, 0, 1], [3, 4, 2])           # the third copy does not fit
    p.check()


@pytest.mark.parametrize("seed", range(6))
def test_long_histories(seed, cuda_device):
    """Random calls one after the other, checked after each."""
    g = torch.Generator().manual_seed(100 + seed)
    page = [1, 4, 16, 7, 8, 3][seed]
    slots = 40
    p = Pool([int(x) for x in torch.randint(0, 6 * page, (12,), generator=g)], page, slots=slots, width=9,
             pages=140, dev=cuda_device, seed=seed, block=(2, 8), dtype=[torch.bfloat16, torch.float32][seed % 2])
    r = lambda n: [int(x) for x in torch.randperm(slots, generator=g)[:n]]
    for step in range(30):
        kind = int(torch.randint(0, 6, (1,), generator=g))
        if kind == 0:
            p.free(r(3))
        elif kind == 1:
            a = r(12)
            p.fork(a[:6], a[6:])
        elif kind == 2:
            a = r(6)
            p.copy(a[:3], a[3:])
        elif kind == 3:
            p.compact()
        else:
            n = 10
            s = r(n)
            room = [9 * page - int(p.m.lens[x]) for x in s]
            p.reserve(s, [min(m, int(x)) for m, x in zip(room, torch.randint(0, 2 * page + 2, (n,), generator=g))])
        p.check()


def test_many_sequences_and_pages(cuda_device):
    """More sequences than one block has threads, more pages than one scan step covers."""
    g = torch.Generator().manual_seed(5)
    n = 1500
    lens = [int(x) for x in torch.randint(0, 20, (n,), generator=g)]
    p = Pool(lens, 4, slots=2 * n, width=6, pages=20000, dev=cuda_device, block=(1, 2), planes=2)
    dst = list(range(n, 2 * n))
    p.fork(list(range(n)), dst)
    p.reserve(dst, [1 + (i % 3) for i in range(n)])
    p.check()
    p.free(list(range(0, n, 2)))
    p.compact()
    p.check()
    p.copy(list(range(1, 400, 2)), list(range(0, 400, 2)))
    p.check()


def test_strided_planes_and_tables(cuda_device):
    """Page data as every second plane of a buffer, tables as views with spare columns."""
    dev = cuda_device
    p = Pool([5, 9, 2], 4, slots=6, width=4, pages=20, dev=dev)
    big = torch.zeros(6, 25, 2, 4, 5, dtype=torch.bfloat16, device=dev)
    p.data = big[::2, 2:22]
    p.data.copy_(p.m.data)
    wide = torch.full((6, 9), 77, dtype=torch.int32, device=dev)
    p.table = wide[:, 3:7]
    p.table.copy_(p.m.table)
    p.fork([0, 1], [3, 4])
    p.reserve([3, 4, 2], [2, 3, 7])
    p.copy([4], [5])
    p.free([0, 1])
    p.compact()
    p.check()
    assert (wide[:, :3] == 77).all() and (wide[:, 7:] == 77).all()
    assert (big[1::2] == 0).all() and (big[:, :2] == 0).all() and (big[:, 22:] == 0).all()


def test_bad_table_entries_are_left_out(cuda_device):
    """A held entry outside the pool: no count, copy or move touches anything for it."""
    dev = cuda_device
    p = Pool([8, 8, 3], 4, slots=6, width=4, pages=12, dev=dev)
    p.table[0, 1] = 99
    p.table[2, 0] = -5
    before = p.data.clone()
    ada.fork_pages(*p.pool, p.ids([0]), p.ids([3]), page_size=4)
    got = ada.reserve_pages(p.data, *p.pool, p.ids([2, 1]), p.ids([1, 1]))
    assert got.tolist() == [0, 1]
    ada.copy_pages(p.data, *p.pool, p.ids([0]), p.ids([4]))
    ada.compact_pages(p.data, *p.pool)
    ada.free_pages(*p.pool, p.ids([0, 3, 4]), page_size=4)
    torch.cuda.synchronize()
    with pytest.raises(ada.KernelError):
        _lib.poll_device_status(dev)
    assert (p.refs >= 0).all() and before.shape == p.data.shape


def test_captured_steps(cuda_device):
    """A fork, a reserve and a free replayed from a graph act on the state they find."""
    dev = cuda_device
    p = Pool([5, 9, 2, 16], 4, slots=8, width=8, pages=60, dev=dev)
    src, dst, new = p.ids([0, 1, 2, 3]), p.ids([4, 5, 6, 7]), p.ids([1, 2, 3, 4])
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ada.fork_pages(*p.pool, src, dst, page_size=4)
        granted = ada.reserve_pages(p.data, *p.pool, dst, new)
        live = ada.compact_pages(p.data, *p.pool)
    p.check()  # a capture runs nothing
    for _ in range(3):
        gr.replay()
        p.m.fork([0, 1, 2, 3], [4, 5, 6, 7])
        want = p.m.reserve([4, 5, 6, 7], [1, 2, 3, 4])
        assert int(live) == p.m.compact()
        assert granted.tolist() == want
        p.check()


def test_refusals(cuda_device):
    dev = cuda_device
    p = Pool([5, 9], 4, slots=4, width=4, pages=12, dev=dev)
    with pytest.raises(TypeError):
        ada.free_pages(*p.pool, p.ids([0]).long(), page_size=4)
    with pytest.raises(ada.ShapeError):
        ada.fork_pages(*p.pool, p.ids([0]), p.ids([1, 2]), page_size=4)
    with pytest.raises(ada.ShapeError):
        ada.reserve_pages(p.data[:, :5], *p.pool, p.ids([0]), p.ids([1]))
    with pytest.raises(ada.ShapeError):
        ada.compact_pages(p.data.transpose(3, 4), *p.pool)
    with pytest.raises(ada.KernelError):
        ada.free_pages(*p.pool, p.ids([0]), page_size=0)
    with pytest.raises(RuntimeError):
        ada.free_pages(p.table.cpu(), p.lens, p.refs, p.ids([0]), page_size=4)
    ada.free_pages(*p.pool, p.ids([]), page_size=4)
    assert ada.reserve_pages(p.data, *p.pool, p.ids([]), p.ids([])).shape == (0,)
    p.check()
