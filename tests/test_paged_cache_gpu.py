"""PagedKVCache over many steps against a plain account of its pages: every
page is either free or in one request's row, whatever the lengths, the rows of
a step and the table's width do."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def paged(device):
    from fp4_fp8_for_torch_mps import paged
    return paged


def new_cache(paged, pages, page, requests, max_len):
    return paged.PagedKVCache(1, pages, page, 1, 16, requests, max_len, torch.bfloat16, "cuda")


def account(c):
    """Free pages and rows together hold each page once, and the head counts the taken ones."""
    head, table = min(int(c.free_head), c.free_pages.numel()), c.block_table[c.block_table >= 0].tolist()
    assert sorted(c.free_pages[head:].tolist() + table) == list(range(c.free_pages.numel()))
    assert head == len(table)


class Plain:
    """The same steps in a loop over requests."""

    def __init__(self, pages, page, requests, max_len):
        self.page, self.cols = page, -(-max_len // page)
        self.free = list(range(pages))
        self.rows = [[-1] * self.cols for _ in range(requests)]
        self.held = [0] * requests
        self.lens = [0] * requests

    def step(self, new, rows):
        cu, kv, pos, slots = [0], [], [], []
        for r, n in enumerate(new):
            n = min(max(n, 0), rows - len(pos))
            for p in range(self.lens[r], self.lens[r] + n):
                col = p // self.page
                if col < self.cols and col >= self.held[r]:
                    assert col == self.held[r]
                    self.rows[r][col] = self.free.pop(0)
                    self.held[r] += 1
                page = self.rows[r][col] if col < self.cols else -1
                pos.append(p)
                slots.append(page * self.page + p % self.page if page >= 0 else -1)
            self.lens[r] += n
            cu.append(cu[-1] + n)
            kv.append(self.lens[r])
        pad = rows - len(pos)
        return cu, kv, pos + [0] * pad, slots + [-1] * pad

    def release(self, r):
        ids = [x for x in self.rows[r] if x >= 0]
        self.free += ids
        self.rows[r], self.held[r], self.lens[r] = [-1] * self.cols, 0, 0


def same_step(c, plain, new, rows):
    s = c.step(i32(new), rows)
    cu, kv, pos, slots = plain.step(new, rows)
    assert s.cu_new.tolist() == cu and s.kv_lens.tolist() == kv == c.lens.tolist()
    assert s.positions.tolist() == pos and s.slots.tolist() == slots
    assert c.block_table.tolist() == plain.rows
    account(c)


def test_requests_past_max_len_take_no_pages(paged):
    c = new_cache(paged, 6, 4, 2, 8)
    for _ in range(40):                                    # 32 tokens beyond the two columns of a row
        s = c.step(i32([1, 0]), 1)
    assert s.slots.tolist() == [-1] and int(c.free_head) == 2
    account(c)
    s = c.step(i32([1, 7]), 8)                             # the other request still finds its pages
    assert s.slots.tolist() == [-1, 8, 9, 10, 11, 12, 13, 14]
    c.release(0)
    c.release(1)
    assert int(c.free_head) == 0 and sorted(c.free_pages.tolist()) == list(range(6))


def test_rows_short_of_the_new_tokens(paged):
    """Tokens without a row are not added: no length, no page, no offset counts them."""
    c = new_cache(paged, 8, 4, 3, 16)
    s = c.step(i32([3, 9, 5]), 7)
    assert s.cu_new.tolist() == [0, 3, 7, 7] and s.kv_lens.tolist() == [3, 4, 0] == c.lens.tolist()
    assert s.slots.tolist() == [0, 1, 2, 4, 5, 6, 7] and int(c.free_head) == 2
    account(c)
    s = c.step(i32([0, 5, 5]), 10)                         # the rest, in another step
    assert s.positions.tolist() == [4, 5, 6, 7, 8, 0, 1, 2, 3, 4] and c.lens.tolist() == [3, 9, 5]
    account(c)


def test_lengths_taken_back(paged):
    """Rejected tokens: lens lowered in place, the request's pages serve the tokens that come instead."""
    c = new_cache(paged, 8, 4, 2, 24)
    plain = Plain(8, 4, 2, 24)
    same_step(c, plain, [6, 3], 9)
    same_step(c, plain, [7, 1], 8)
    c.lens -= i32([6, 1])
    plain.lens = [7, 3]
    same_step(c, plain, [3, 6], 9)
    c.lens[0] = 0
    plain.lens[0] = 0
    same_step(c, plain, [13, 0], 13)
    for r in (0, 1):
        c.release(r)
    assert int(c.free_head) == 0


def test_pool_runs_short(paged):
    c = new_cache(paged, 3, 4, 2, 16)
    s = c.step(i32([9, 6]), 15)
    assert s.slots[-6:].tolist() == [-1] * 6 and int(c.free_head) == 5
    account_head = c.block_table[c.block_table >= 0]
    assert account_head.tolist() == [0, 1, 2]
    c.release(0)
    s = c.step(i32([1, 3]), 4)                             # a new page for the part that still has room; the lost tokens stay lost
    assert s.positions.tolist() == [0, 6, 7, 8] and s.slots.tolist() == [0, -1, -1, 4]
    c.release(0)
    c.release(1)
    assert int(c.free_head) == 0 and sorted(c.free_pages.tolist()) == [0, 1, 2]


@pytest.mark.parametrize("page,requests", [(1, 3), (4, 7), (16, 40), (3, 700)])
def test_random_steps(paged, page, requests):
    r = random.Random(page * 1000 + requests)
    max_len = 5 * page + 2
    pages = requests * -(-max_len // page)
    c, plain = new_cache(paged, pages, page, requests, max_len), Plain(pages, page, requests, max_len)
    for i in range(25):
        new = [r.choice((0, 1, 1, r.randint(0, 2 * page + 1), -2)) for _ in range(requests)]
        total = sum(max(n, 0) for n in new)
        same_step(c, plain, new, max(0, total + r.choice((0, 0, 3, -1, -total // 2))))
        if i % 3 == 0:
            back = [r.randint(0, min(n, page + 1)) if r.random() < 0.3 else 0 for n in plain.lens]
            c.lens -= i32(back)
            plain.lens = [n - b for n, b in zip(plain.lens, back)]
        if i % 4 == 1:
            for q in r.sample(range(requests), min(requests, 3)):
                c.release(q)
                plain.release(q)
            account(c)


def test_captured_steps(paged):
    """Steps replayed from a graph move the bookkeeping on as eager steps do, also past max_len and after lens went back."""
    c, plain = new_cache(paged, 12, 4, 3, 12), Plain(12, 4, 3, 12)
    same_step(c, plain, [5, 0, 9], 14)
    new = i32([1, 1, 1])
    state = [t.clone() for t in (c.lens, c.free_head, c.block_table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s = c.step(new, 3)
    assert all(torch.equal(a, b) for a, b in zip(state, (c.lens, c.free_head, c.block_table)))
    for i in range(9):
        graph.replay()
        cu, kv, pos, slots = plain.step([1, 1, 1], 3)
        assert s.slots.tolist() == slots and s.positions.tolist() == pos and c.lens.tolist() == kv
        account(c)
        if i == 4:
            c.lens -= i32([3, 2, 0])
            plain.lens = [plain.lens[0] - 3, plain.lens[1] - 2, plain.lens[2]]
