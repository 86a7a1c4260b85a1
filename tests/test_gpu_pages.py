"""Page bookkeeping on the GPU against the same rules in plain Python, entry for entry and byte for byte."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma

pytestmark = pytest.mark.gpu


class Pool:
    """The rules in plain Python: lowest free page first, in the order of the requests."""

    def __init__(self, rows, width, pages, bs, planes):
        self.table = [[-1] * width for _ in range(rows)]
        self.lens = [0] * rows
        self.refs = [0] * pages
        self.bs, self.width = bs, width
        self.planes = [p.clone() for p in planes]

    def take(self):
        for p, n in enumerate(self.refs):
            if n == 0:
                self.refs[p] = 1
                return p
        return -1

    def grow(self, rows, more):
        missing = 0
        for r, n in zip(rows, more):
            if not 0 <= r < len(self.table) or n <= 0:
                continue
            have, end = -(-self.lens[r] // self.bs), min(self.lens[r] + n, self.width * self.bs)
            for j in range(have, -(-end // self.bs)):
                p = self.take()
                if p < 0:
                    end = j * self.bs
                    break
                self.table[r][j] = p
            end = max(end, self.lens[r])
            missing += self.lens[r] + n - end
            self.lens[r] = end
        return missing

    def fork(self, parents, children):
        missing, moved = 0, []
        fresh = []
        for p, c in zip(parents, children):
            full, rest = divmod(self.lens[p], self.bs)
            to = -1
            if rest:
                to = self.take()
                missing += to < 0
                if to >= 0:
                    moved.append((self.table[p][full], to))
            fresh.append((p, c, full, to))
        for p, c, full, to in fresh:
            row = self.table[p][:full] + [to] + [-1] * self.width
            self.table[c] = row[: self.width]
            for q in self.table[p][:full]:
                self.refs[q] += 1
            self.lens[c] = self.lens[p] if to >= 0 else full * self.bs
        self.move(moved)
        return missing

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.table):
                for q in self.table[r]:
                    if q >= 0:
                        self.refs[q] -= 1
                self.table[r] = [-1] * self.width
                self.lens[r] = 0

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        src = [p for p, n in enumerate(self.refs) if n > 0 and p >= live]
        dst = [p for p, n in enumerate(self.refs) if n <= 0 and p < live]
        self.move(list(zip(src, dst)))
        to = dict(zip(src, dst))
        self.table = [[to.get(q, q) for q in row] for row in self.table]
        for s, d in zip(src, dst):
            self.refs[d], self.refs[s] = self.refs[s], 0
        return live

    def move(self, pairs):
        for plane in self.planes:
            for s, d in pairs:
                plane[d] = plane[s]


class Device:
    def __init__(self, pool, offset=0):
        self.table = torch.tensor(pool.table, dtype=torch.int32).cuda()
        self.lens = torch.tensor(pool.lens, dtype=torch.int32).cuda()
        room = torch.zeros(len(pool.refs) + offset, dtype=torch.int32, device="cuda")
        self.refs = room[offset:]
        self.planes = [p.cuda() for p in pool.planes]

    def same(self, pool):
        assert self.table.cpu().tolist() == pool.table
        assert self.lens.cpu().tolist() == pool.lens
        assert self.refs.cpu().tolist() == pool.refs
        for a, b in zip(self.planes, pool.planes):
            assert torch.equal(a.cpu().contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def planes_of(pages, g, layers=2):
    made = []
    for _ in range(layers):
        made.append(torch.randint(-127, 128, (pages, 2, 64, 16), generator=g).to(torch.int8))
        made.append(torch.randn((pages, 3), generator=g))  # 12-byte pages
        made.append(torch.randn((pages, 5, 8), generator=g).to(torch.bfloat16))
        made.append(torch.randint(0, 255, (pages, 7), generator=g).to(torch.uint8))  # 7-byte pages
    return made


@pytest.mark.parametrize("pages,rows,width,bs,offset", [(40, 6, 9, 16, 0), (300, 30, 20, 4, 1), (20000, 50, 60, 16, 0), (9000, 20, 400, 1, 3)])
def test_a_schedule(pages, rows, width, bs, offset):
    """Requests come, are forked, grow, end; the pool is compacted now and then and runs out at times."""
    g = torch.Generator().manual_seed(pages)
    pool = Pool(rows, width, pages, bs, planes_of(pages, g) if pages < 10000 else [torch.randn((pages, 9), generator=g)])
    dev = Device(pool, offset)
    for step in range(25):
        pick = torch.randperm(rows, generator=g).tolist()
        empty = [r for r in pick if pool.lens[r] == 0]
        held = [r for r in pick if pool.lens[r] > 0]
        what = step % 5
        if what in (0, 1) or not held:
            who = pick[: max(1, rows // 2)]
            more = torch.randint(0, max(2, width * bs // 2), (len(who),), generator=g).tolist()
            got = ma.kv_pages_grow(dev.table, dev.lens, i32(who), i32(more), dev.refs, bs)
            assert int(got) == pool.grow(who, more)
        elif what == 2:
            children = empty[: rows // 3]
            parents = [held[int(i)] for i in torch.randint(0, len(held), (len(children),), generator=g)]
            got = ma.kv_pages_fork(dev.table, dev.lens, i32(parents), i32(children), dev.refs, dev.planes, bs)
            assert int(got) == pool.fork(parents, children)
        elif what == 3:
            who = held[: max(1, len(held) // 2)]
            ma.kv_pages_free(dev.table, dev.lens, i32(who + [-1, rows, who[0]]), dev.refs)
            pool.free(who)
        else:
            live = ma.kv_pages_compact(dev.table, dev.refs, dev.planes)
            assert int(live) == pool.compact()
        dev.same(pool)


def test_more_requests_than_one_launch_plans():
    g = torch.Generator().manual_seed(1)
    rows, pages, bs = 9001, 12000, 4
    pool = Pool(2 * rows, 2, pages, bs, [torch.randn((pages, 4), generator=g)])
    dev = Device(pool)
    who = list(range(rows))
    more = torch.randint(0, 7, (rows,), generator=g).tolist()
    # the plain pool's search for a free page is linear: give the pages out in its order directly
    nxt = 0
    missing = 0
    for r, n in zip(who, more):
        end = n
        for j in range(-(-n // bs)):
            if nxt == pages:
                end = j * bs
                break
            pool.table[r][j] = nxt
            pool.refs[nxt] = 1
            nxt += 1
        pool.lens[r] = end
        missing += n - end
    assert int(ma.kv_pages_grow(dev.table, dev.lens, i32(who), i32(more), dev.refs, bs)) == missing
    dev.same(pool)
    gone = who[: rows // 2]
    ma.kv_pages_free(dev.table, dev.lens, i32(gone), dev.refs)
    pool.free(gone)
    dev.same(pool)
    parents = [r for r in who[rows // 2:] if pool.lens[r]]
    children = list(range(rows, rows + len(parents)))
    free = iter([p for p, n in enumerate(pool.refs) if n == 0])
    pool.take = lambda: next(free, -1)
    fork = pool.fork(parents, children)
    for row in children:
        for q in pool.table[row]:
            if q >= 0 and pool.refs[q] == 0:
                pool.refs[q] = 1
    assert int(ma.kv_pages_fork(dev.table, dev.lens, i32(parents), i32(children), dev.refs, dev.planes, bs)) == fork
    dev.same(pool)


@pytest.mark.parametrize("layers", [1, 40])
def test_copy(layers):
    """More planes than one launch takes, pages of a strided tensor, pairs out of range."""
    g = torch.Generator().manual_seed(layers)
    pages = 50
    planes = planes_of(pages, g, layers)
    wide = torch.randn((pages, 4, 32), generator=g)
    dev = [p.cuda() for p in planes]
    dwide = wide.cuda()
    src, dst = [3, -1, 7, 50, 9, 3], [10, 11, -5, 12, 49, 0]
    ma.kv_pages_copy(dev + [dwide[:, 1:3]], i32(src), i32(dst))
    for p in planes:
        for s, d in ((3, 10), (9, 49), (3, 0)):
            p[d] = p[s]
    for s, d in ((3, 10), (9, 49), (3, 0)):
        wide[d, 1:3] = wide[s, 1:3]
    for a, b in zip(dev + [dwide], planes + [wide]):
        assert torch.equal(a.cpu(), b)


def test_empty_requests():
    refs, table, lens = i32([1, 0, 2]), i32([[0, 2]]), i32([20])
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    plane = torch.arange(12.0).view(3, 4).cuda()
    assert int(ma.kv_pages_fork(table, lens, none, none, refs, [plane], 16)) == 0
    assert int(ma.kv_pages_grow(table, lens, none, none, refs, 16)) == 0
    ma.kv_pages_free(table, lens, none, refs)
    ma.kv_pages_copy([plane], none, none)
    assert int(ma.kv_pages_compact(table, refs, [])) == 2
    assert table.tolist() == [[0, 1]] and refs.tolist() == [1, 2, 0]
    assert torch.equal(plane.cpu(), torch.arange(12.0).view(3, 4))


def test_forked_rows_do_not_share_what_they_write():
    """A prompt is written, forked, and each child appends its own tokens: shared pages stay as they were."""
    g = torch.Generator().manual_seed(2)
    nh, hd, bs, pages = 2, 64, 16, 12
    kc = torch.zeros((pages, nh, hd, bs), dtype=torch.int8, device="cuda")
    vc, ks, vs = kc.clone(), torch.zeros((pages, nh), device="cuda"), torch.zeros((pages, nh), device="cuda")
    table, lens = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    ma.kv_pages_grow(table, lens, i32([0]), i32([37]), refs, bs)
    x = torch.randn((37, nh, hd), generator=g).half().cuda()
    ma.kv_append_block_scaled(x, x, kc, vc, ks, vs, table[:1], lens[:1], i32([0, 37]))
    ma.kv_pages_fork(table, lens, i32([0, 0]), i32([1, 2]), refs, [kc, vc, ks, vs], bs)
    before = kc.clone()
    ma.kv_pages_grow(table, lens, i32([1, 2]), i32([1, 1]), refs, bs)
    y = torch.randn((2, nh, hd), generator=g).half().cuda() * 0.1
    ma.kv_append_block_scaled(y, y, kc, vc, ks, vs, table[1:], lens[1:])
    assert refs.tolist()[:5] == [3, 3, 1, 1, 1] and table.tolist() == [[0, 1, 2, -1], [0, 1, 3, -1], [0, 1, 4, -1]]
    assert torch.equal(kc[:3], before[:3]) and lens.tolist() == [37, 38, 38]
    assert torch.equal(kc[3, ..., :5], kc[2, ..., :5]) and not torch.equal(kc[3, ..., 5], kc[4, ..., 5])
    # what the children see of the prompt is what its own row sees
    q = torch.randn((1, 4, hd), generator=g).half().cuda()
    a = ma.paged_attention_block_scaled(q, kc, vc, ks, vs, table[:1], i32([37]))
    b = ma.paged_attention_block_scaled(q, kc, vc, ks, vs, table[1:2], i32([37]))
    assert torch.equal(a, b)
