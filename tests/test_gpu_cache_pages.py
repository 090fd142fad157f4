"""A cache's pages: the next batch's tables (vtq_pages_reorder_device), closing up (vtq_pages_compact_device) and copies
(vtq_pages_copy_device, vtq_kv8_pages_copy_device), against the same done one sequence, one page after another."""
import random

import pytest
import torch

import vtq
from serving import TAGS, TYPES, stream

pytestmark = pytest.mark.gpu


def _ints(x, *shape):
    return torch.tensor(x, dtype=torch.int32).reshape(shape).cuda()


def reorder(n_pages, page, refs, table, lens, parents, grow):
    """(new refs, new table, new lens, copies, missing), one sequence after another."""
    most = len(table[0]) if table else 0
    free = [p for p, r in enumerate(refs) if r == 0]
    new_refs = list(refs)
    is_page = lambda p: 0 <= p < n_pages  # noqa: E731
    for row in table:
        for p in row:
            if is_page(p):
                new_refs[p] -= 1
    rows, new_lens, copies, missing, seen = [], [], [], 0, set()
    for i, parent in enumerate(parents):
        has = 0 <= parent < len(table)
        old = table[parent] if has else [-1] * most
        n = min(max(lens[parent], 0), most * page) if has else 0
        whole, wanted = n // page, -(-(n + max(grow[i], 0)) // page)
        needed = min(wanted, most)
        missing += wanted - needed
        row = [p if is_page(p) else -1 for p in old[:whole]]
        if has and parent not in seen:
            while len(row) < needed and is_page(old[len(row)]) and refs[old[len(row)]] == 1:
                row.append(old[len(row)])
        seen.add(parent)
        for p in row:
            if is_page(p):
                new_refs[p] += 1
        while len(row) < needed:
            j = len(row)
            if free:
                p = free.pop(0)
                new_refs[p] += 1
                if j == whole and n % page and is_page(old[j]):
                    copies.append((old[j], p, n % page))
                row.append(p)
            else:
                missing += 1
                row.append(-1)
        rows.append(row + [-1] * (most - len(row)))
        new_lens.append(n)
    return new_refs, rows, new_lens, copies, missing


def run_reorder(ctx, n_pages, page, refs, table, lens, parents, grow, wait=True, most=None):
    most = len(table[0]) if most is None else most
    b, o = len(table), len(parents)
    st = dict(refs=_ints(refs, -1), table=_ints(table, b, most), lens=_ints(lens, -1), parents=_ints(parents, -1),
              grow=None if grow is None else _ints(grow, -1))
    new = dict(refs=torch.full((n_pages,), 77, dtype=torch.int32, device="cuda"),
               table=torch.full((o, most), 77, dtype=torch.int32, device="cuda"),
               lens=torch.full((o,), 77, dtype=torch.int32, device="cuda"),
               copies=torch.full((o, 3), 77, dtype=torch.int32, device="cuda"),
               info=torch.full((2,), 77, dtype=torch.int32, device="cuda"))
    need = ctx.pages_reorder_workspace(n_pages, b, o)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")

    def call():
        ctx.pages_reorder_device(n_pages, page, most, st["refs"].data_ptr(), b, st["table"].data_ptr(),
                                 st["lens"].data_ptr(), o, st["parents"].data_ptr(),
                                 None if grow is None else st["grow"].data_ptr(), new["refs"].data_ptr(),
                                 new["table"].data_ptr(), new["lens"].data_ptr(), new["copies"].data_ptr(),
                                 new["info"].data_ptr(), ws.data_ptr(), need, stream())

    call()
    torch.cuda.synchronize()
    assert (ws[need:] == 255).all()
    return st, new, call, ws


def check_reorder(new, want):
    refs, rows, lens, copies, missing = want
    assert new["info"].tolist() == [len(copies), missing]
    assert new["lens"].tolist() == lens
    assert new["table"].tolist() == rows
    assert new["copies"].tolist() == [list(c) for c in copies] + [[-1] * 3] * (len(new["copies"]) - len(copies))
    assert new["refs"].tolist() == refs


def a_batch(rng, n_pages, page, batch, most, shared=0.3):
    """Consistent tables: sequences with pages of their own, some sharing their first ones."""
    free = list(range(n_pages))
    rng.shuffle(free)
    table, lens, refs = [], [], [0] * n_pages
    for b in range(batch):
        n = rng.randint(0, most * page)
        row = []
        if table and rng.random() < shared:
            other = rng.randrange(len(table))
            same = rng.randint(0, min(lens[other], n) // page)
            row = list(table[other][:same])
        held = min(most, -(-n // page) + (rng.randint(0, 2) if rng.random() < 0.5 else 0))
        while len(row) < held and free:
            row.append(free.pop())
        n = min(n, len(row) * page)
        for p in row:
            refs[p] += 1
        table.append(row + [-1] * (most - len(row)))
        lens.append(n)
    return table, lens, refs


@pytest.mark.parametrize("seed", range(12))
def test_reorder(ctx, seed):
    rng = random.Random(seed)
    page, most, batch = rng.choice([8, 16, 64]), rng.choice([1, 3, 9, 40]), rng.choice([1, 2, 5, 17, 70])
    n_pages = int(batch * most * rng.choice([0.4, 1.0, 2.0])) + rng.choice([0, 3, 5000])
    n_pages = max(n_pages, 1)
    table, lens, refs = a_batch(rng, n_pages, page, batch, most)
    out = rng.choice([batch, 1, 2 * batch, batch + 3])
    parents = [rng.randint(-1, batch) for _ in range(out)]  # -1 and batch: empty ones
    grow = [rng.choice([0, 1, 1, page, 3 * page, -5, most * page]) for _ in range(out)]
    st, new, call, ws = run_reorder(ctx, n_pages, page, refs, table, lens, parents, grow)
    check_reorder(new, reorder(n_pages, page, refs, table, lens, parents, grow))
    # again: nothing that the call read has changed
    ws.fill_(0)
    before = {k: v.clone() for k, v in new.items()}
    call()
    torch.cuda.synchronize()
    assert all(torch.equal(before[k], new[k]) for k in new)
    assert st["refs"].tolist() == refs and st["table"].tolist() == table and st["lens"].tolist() == lens


def test_counts_stay_those_of_the_tables_over_many_steps(ctx):
    rng = random.Random(5)
    page, most, n_pages = 16, 6, 200
    table, lens, refs = a_batch(rng, n_pages, page, 12, most)
    for step in range(25):
        out = rng.randint(1, 14)
        parents = [rng.randint(-1, len(table) - 1) for _ in range(out)]
        grow = [rng.randint(0, 20) for _ in range(out)]
        _, new, _, _ = run_reorder(ctx, n_pages, page, refs, table, lens, parents, grow)
        want = reorder(n_pages, page, refs, table, lens, parents, grow)
        check_reorder(new, want)
        refs, table, lens, _, missing = want
        flat = [p for row in table for p in row if p >= 0]
        assert [flat.count(p) for p in range(n_pages)] == refs
        lens = [min(n + max(g, 0), most * page) if not missing else n for n, g in zip(lens, grow)]
        for row, n in zip(table, lens):  # no two sequences write one page
            for j in range(-(-n // page)):
                assert missing or row[j] >= 0


def test_the_edges_of_a_reorder(ctx):
    # nothing at all; no old batch; all sequences end; no pages
    _, new, _, _ = run_reorder(ctx, 5, 16, [0, 1, 0, 2, 0], [], [], [], [], most=4)
    assert new["info"].tolist() == [0, 0] and new["refs"].tolist() == [0, 1, 0, 2, 0]
    _, new, _, _ = run_reorder(ctx, 5, 16, [0, 1, 0, 2, 0], [], [], [-1, 3], [33, 0], most=4)
    assert new["table"].tolist() == [[0, 2, 4, -1], [-1] * 4] and new["info"].tolist() == [0, 0]
    _, new, _, _ = run_reorder(ctx, 5, 16, [1, 1, 0, 2, 0], [[0, 1], [3, -1]], [20, 16], [], [])
    assert new["refs"].tolist() == [0, 0, 0, 1, 0] and new["info"].tolist() == [0, 0]
    _, new, _, _ = run_reorder(ctx, 0, 16, [], [[-1, 7]], [5], [0, 0], [40, 0])
    assert new["table"].tolist() == [[-1, -1], [-1, -1]] and new["info"].tolist() == [0, 1 + 3 + 0]
    # no growth asked for: a fork of a part-filled page
    _, new, _, _ = run_reorder(ctx, 3, 16, [1, 0, 0], [[0, -1]], [5], [0, 0, 0], None)
    assert new["table"].tolist() == [[0, -1], [1, -1], [2, -1]] and new["info"].tolist() == [2, 0]
    assert new["copies"].tolist() == [[0, 1, 5], [0, 2, 5], [-1] * 3]
    # pages run out between two forks: the second has none to copy to
    _, new, _, _ = run_reorder(ctx, 2, 16, [1, 0], [[0, -1]], [5], [0, 0, 0], None)
    assert new["table"].tolist() == [[0, -1], [1, -1], [-1, -1]] and new["info"].tolist() == [1, 1]
    # numbers that are no pages hold nothing; lengths past the table are cut
    st = ([0, 1, 0, 0], [[9, 1, -4], [2 ** 31 - 1, -1, -1]], [40, 2 ** 31 - 1], [0, 1], [1, 0])
    _, new, _, _ = run_reorder(ctx, 4, 16, *st)
    check_reorder(new, reorder(4, 16, *st))


def test_many_sequences_and_pages(ctx):
    rng = random.Random(2)
    page, most, batch, n_pages = 16, 4, 3000, 20000
    table, lens, refs = a_batch(rng, n_pages, page, batch, most)
    parents = [rng.randint(-1, batch - 1) for _ in range(batch)]
    grow = [rng.randint(0, 30) for _ in range(batch)]
    _, new, _, _ = run_reorder(ctx, n_pages, page, refs, table, lens, parents, grow)
    check_reorder(new, reorder(n_pages, page, refs, table, lens, parents, grow))


def compact(refs, entries, prefix, page):
    live = [p for p, r in enumerate(refs) if r > 0]
    n = len(live)
    high, low = [p for p in live if p >= n], [p for p in range(n) if refs[p] <= 0]
    goes = dict(zip(high, low))
    new_refs = [0] * len(refs)
    for p in live:
        new_refs[goes.get(p, p)] = refs[p]
    move = lambda p: goes.get(p, p) if 0 <= p < len(refs) else -1  # noqa: E731
    return new_refs, [move(p) for p in entries], [move(p) for p in prefix], [(h, l, page) for h, l in zip(high, low)], n


@pytest.mark.parametrize("n_pages", [0, 1, 2, 3, 64, 255, 1000, 4095, 4096, 4097, 8192, 20011])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 0.97, 1.0])
def test_compact(ctx, n_pages, share):
    _compact(ctx, n_pages, share, 700)


@pytest.mark.parametrize("n_pages,places", [(0, 5), (3, 0), (100, 1 << 16), (4096, 1 << 16), (4096, (1 << 16) + 1),
                                            (37, 100000), (0, 100000)])
def test_compact_of_many_places(ctx, n_pages, places):
    _compact(ctx, n_pages, 0.6, places)


def _compact(ctx, n_pages, share, places):
    rng = random.Random(n_pages)
    refs = [rng.randint(1, 5) if rng.random() < share else 0 for _ in range(n_pages)]
    entries = [rng.randint(-2, n_pages + 1) for _ in range(places)]
    prefix = [rng.randint(-2, n_pages + 1) for _ in range(9)]
    want = compact(refs, entries, prefix, 32)
    r, e, x = _ints(refs, -1), _ints(entries, -1), _ints(prefix, -1)
    new_r, new_e, new_x = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for n in (n_pages, places, 9))
    copies = torch.full((n_pages // 2 + 1, 3), 77, dtype=torch.int32, device="cuda")  # one row to spare
    info = torch.full((2,), 77, dtype=torch.int32, device="cuda")
    need = ctx.pages_compact_workspace(n_pages)
    ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    ctx.pages_compact_device(n_pages, 32, r.data_ptr(), places, e.data_ptr(), new_r.data_ptr(), new_e.data_ptr(),
                             copies.data_ptr(), info.data_ptr(), ws.data_ptr(), need, stream(), n_prefix=9,
                             prefix_pages_ptr=x.data_ptr(), new_prefix_pages_ptr=new_x.data_ptr())
    torch.cuda.synchronize()
    assert (ws[need:] == 255).all() and (copies[-1] == 77).all()
    # an entry that names a page not in use keeps a number that may mean another page now: only those in use are compared
    assert info.tolist() == [len(want[3]), want[4]]
    assert new_r.tolist() == want[0]
    assert copies[:n_pages // 2].tolist() == [list(c) for c in want[3]] + [[-1] * 3] * (n_pages // 2 - len(want[3]))
    assert new_e.tolist() == want[1] and new_x.tolist() == want[2]


# ------------------------------------------------------------------ copies

def _expect_copies(x, copies, page, slot_dim, block=1):
    """x with pages first, and the slots (or their blocks) in dimension slot_dim."""
    y = x.clone()
    for source, target, slots in copies:
        if 0 <= source < x.shape[0] and 0 <= target < x.shape[0]:
            n = -(-min(max(slots, 0), page) // block)
            y[target].narrow(slot_dim - 1, 0, n).copy_(x[source].narrow(slot_dim - 1, 0, n))
    return y


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("layers,kv_heads,head_dim,page,n_pages,order", [
    (1, 1, 16, 16, 7, "heads"), (3, 2, 64, 16, 40, "heads"), (2, 3, 80, 32, 30, "slots"), (1, 8, 128, 128, 24, "heads"),
    (2, 4, 256, 64, 20, "major"), (22, 4, 64, 16, 60, "heads")])
def test_copies(ctx, cache, layers, kv_heads, head_dim, page, n_pages, order):
    g = torch.Generator().manual_seed(n_pages)
    shape = {"heads": (layers, n_pages, kv_heads, page, head_dim), "slots": (layers, n_pages, page, kv_heads, head_dim),
             "major": (layers, kv_heads, n_pages, page, head_dim)}[order]
    dim = {"heads": 2, "slots": 1, "major": 2}[order]  # of the slots, pages first
    pages_first = lambda t: t.transpose(0, 1) if order == "major" else t  # noqa: E731
    dtype = {"e4m3": torch.uint8}.get(cache) or TYPES[cache]
    k, v = ((torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) if cache == "e4m3"
             else torch.randn(shape, generator=g).to(dtype)).cuda() for _ in range(2))
    scales = [torch.randint(0, 256, (layers, n_pages, kv_heads, page // 16), generator=g, dtype=torch.uint8).cuda()
              for _ in range(2)]
    at = k[0].stride()
    s = dict(zip({"heads": ("page_stride", "head_stride", "slot_stride"), "slots": ("page_stride", "slot_stride", "head_stride"),
                  "major": ("head_stride", "page_stride", "slot_stride")}[order], at))
    if cache == "e4m3":
        desc = vtq.Kv8Cache(k.data_ptr(), v.data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), n_pages, page, kv_heads,
                            head_dim, block=16, **s)
    else:
        desc = vtq.KvCache(TAGS[cache], k.data_ptr(), v.data_ptr(), n_pages, page, kv_heads, head_dim, **s)
    order_ = torch.randperm(n_pages, generator=g).tolist()
    half = n_pages // 2
    rng = random.Random(3)
    copies = [(order_[rng.randrange(half)], order_[half + i], rng.choice([0, 1, 15, 16, 17, page - 1, page, page + 9, -3]))
              for i in range(n_pages - half)]
    copies[-1] = (copies[-1][0], n_pages, 5)
    copies[-2] = (-1, copies[-2][1], 5)
    for valid in (0, 2, len(copies), None, len(copies) + 50):
        want = []
        rows = copies if valid is None else copies[:valid]
        for t in (k, v):
            want.append([_expect_copies(pages_first(t[i]), rows, page, dim) for i in range(layers)])
        want_s = [[_expect_copies(t[i], rows, page, 2, 16) for i in range(layers)] for t in scales]
        count = None if valid is None else _ints([valid], -1)
        ctx.pages_copy_device(desc, layers, k.stride(0), _ints(copies, -1, 3).data_ptr(), len(copies),
                              None if count is None else count.data_ptr(), stream(),
                              scale_layer_stride=scales[0].stride(0) if cache == "e4m3" else 0)
        torch.cuda.synchronize()
        for t, w in zip((k, v), want):
            assert all(torch.equal(pages_first(t[i]), w[i]) for i in range(layers))
        if cache == "e4m3":
            for t, w in zip(scales, want_s):
                assert all(torch.equal(t[i], w[i]) for i in range(layers))


def test_copies_past_32_bits(ctx):
    d, page, n_pages = 64, 64, (1 << 32) // (64 * 64) + 100
    k, v = (torch.zeros(n_pages, 1, page, d, dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = torch.zeros(2, n_pages, 1, 4, dtype=torch.uint8, device="cuda")
    k[-1], v[-2], scales[:, -1] = 9, 8, 7
    desc = vtq.Kv8Cache(k.data_ptr(), v.data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), n_pages, page, 1, d)
    copies = _ints([[n_pages - 1, 3, 20], [n_pages - 2, n_pages - 3, 64]], 2, 3)
    ctx.pages_copy_device(desc, 1, 0, copies.data_ptr(), 2, None, stream())
    torch.cuda.synchronize()
    assert (k[3, 0, :20] == 9).all() and not k[3, 0, 20:].any() and (v[-3] == 8).all()
    assert scales[:, 3, 0].tolist() == [[7, 7, 0, 0]] * 2


def test_a_captured_step_follows_its_lists(ctx):
    rng = random.Random(8)
    page, most, n_pages, batch = 16, 5, 100, 6
    table, lens, refs = a_batch(rng, n_pages, page, batch, most)
    parents = [rng.randrange(batch) for _ in range(batch)]
    st, new, call, ws = run_reorder(ctx, n_pages, page, refs, table, lens, parents, [1] * batch)
    k, v = (torch.randn(2, n_pages, 2, page, 32, device="cuda").bfloat16() for _ in range(2))
    desc = vtq.KvCache(vtq.BF16, k.data_ptr(), v.data_ptr(), n_pages, page, 2, 32)

    def step():
        call()
        ctx.pages_copy_device(desc, 2, k.stride(0), new["copies"].data_ptr(), batch, new["info"].data_ptr(), stream())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx_stream = stream()
        assert ctx_stream
        step()
    for i in range(4):
        parents = [rng.randrange(batch) for _ in range(batch)]
        st["parents"].copy_(torch.tensor(parents, dtype=torch.int32))
        ws.fill_(255)
        before = k.clone(), v.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = reorder(n_pages, page, refs, table, lens, parents, [1] * batch)
        check_reorder(new, want)
        for t, old in zip((k, v), before):
            for layer in range(2):
                assert torch.equal(t[layer], _expect_copies(old[layer], want[3], page, 2))
