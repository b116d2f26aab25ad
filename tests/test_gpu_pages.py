"""The page operations of a paged cache (b2a_pages_reserve / fork / free / compact) against a plain
sequential model: table, counts, contents and returned numbers are whole numbers and must be equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Model:
    def __init__(self, rng, n_seq, max_pages, num_pages, page, layers=2, words=16, share=0.3, fill=0.6):
        self.page = page
        self.table = np.full((n_seq, max_pages), -1, np.int32)
        self.lens = np.zeros(n_seq, np.int32)
        free = list(rng.permutation(num_pages))
        for b in range(n_seq):
            used = int(rng.integers(0, int(max_pages * fill) + 1))
            src = int(rng.integers(0, b)) if b and rng.random() < share else -1
            for i in range(used):
                if src >= 0 and self.table[src, i] >= 0:
                    self.table[b, i] = self.table[src, i]
                elif free:
                    self.table[b, i] = free.pop()
                else:
                    used = i
                    break
            self.lens[b] = max(0, used * page - int(rng.integers(0, page))) if used else 0
        self.refs = np.zeros(num_pages, np.int32)
        np.add.at(self.refs, self.table[self.table >= 0], 1)
        self.pages = rng.integers(0, 256, (layers, num_pages, words), dtype=np.uint8)
        self.counts = np.zeros(2, np.int32)

    def fork(self, parents):
        after = np.where(parents[:, None] >= 0, self.table[np.maximum(parents, 0)], -1)
        self.refs[:] = 0
        np.add.at(self.refs, after[after >= 0], 1)
        self.table = after.astype(np.int32)

    def free(self, keep_from, keep_to):
        for b, i in zip(*np.nonzero(self.table >= 0)):
            lo = 0 if keep_from is None else keep_from[b]
            if not (i * self.page < keep_to[b] and (i + 1) * self.page > lo):
                self.refs[self.table[b, i]] -= 1
                self.table[b, i] = -1

    def reserve(self, lens, new):
        refs0, want = self.refs.copy(), []
        for b in range(len(lens)):
            if new[b] > 0:
                for i in range(lens[b] // self.page, (lens[b] + new[b] - 1) // self.page + 1):
                    if self.table[b, i] < 0 or refs0[self.table[b, i]] > 1:
                        want.append((b, i))
        free = np.nonzero(refs0 == 0)[0]
        if len(want) > len(free):
            self.counts[:] = 0, len(want) - len(free)
            return
        for (b, i), p in zip(want, free):
            old = self.table[b, i]
            if old >= 0:
                self.pages[:, p] = self.pages[:, old]
                self.refs[old] -= 1
            self.refs[p], self.table[b, i] = 1, p
        self.counts[:] = len(want), 0

    def compact(self):
        n = int((self.refs > 0).sum())
        src = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(n) if self.refs[p] == 0]
        for s, d in zip(src, dst):
            self.pages[:, d] = self.pages[:, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.table[self.table == s] = d
        self.counts[:] = n, len(src)

    def device(self):
        import torch
        return {k: torch.from_numpy(getattr(self, k).copy()).cuda() for k in ("table", "refs", "pages", "counts", "lens")}

    def check(self, t):
        for k in ("table", "refs", "pages", "counts"):
            np.testing.assert_array_equal(t[k].cpu().numpy(), getattr(self, k), err_msg=k)


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


SHAPES = [(1, 1, 3, 16), (3, 5, 12, 16), (40, 33, 900, 48), (1500, 3, 5000, 16), (7, 700, 6000, 32), (2100, 9, 20011, 64)]


@pytest.mark.parametrize("n_seq,max_pages,num_pages,page", SHAPES)
def test_a_history_of_operations(ctx, n_seq, max_pages, num_pages, page):
    import b200attn
    rng = np.random.default_rng(n_seq * 31 + max_pages)
    m = Model(rng, n_seq, max_pages, num_pages, page, words=16 * int(rng.integers(1, 5)))
    t = m.device()
    room = max_pages * page
    for step in range(3):
        new = np.minimum(rng.integers(0, 3 * page, n_seq), room - m.lens).astype(np.int32)
        new[rng.random(n_seq) < 0.3] = 0
        b200attn.pages_reserve(ctx, t["table"], t["refs"], t["lens"], _dev(new), t["pages"], page, t["counts"])
        m.reserve(m.lens, new)
        m.check(t)
        keep_to = np.maximum(0, m.lens - rng.integers(0, 2 * page, n_seq)).astype(np.int32)
        keep_from = None if step == 1 else (keep_to * rng.random(n_seq) * 0.5).astype(np.int32)
        b200attn.pages_free(ctx, t["table"], t["refs"], None if keep_from is None else _dev(keep_from), _dev(keep_to), page)
        m.free(keep_from, keep_to)
        m.check(t)
        parents = rng.integers(-1, n_seq, n_seq).astype(np.int32)
        parents[rng.random(n_seq) < 0.5] = -1 if step == 2 else 0
        stay = rng.random(n_seq) < 0.3
        parents[stay] = np.nonzero(stay)[0]
        b200attn.pages_fork(ctx, t["table"], t["refs"], _dev(parents))
        m.fork(parents)
        m.check(t)
        m.lens = np.where(parents >= 0, np.minimum(m.lens, keep_to)[np.maximum(parents, 0)], 0).astype(np.int32)
        t["lens"].copy_(_dev(m.lens))
        b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"], t["counts"])
        m.compact()
        m.check(t)
    ctx.check_device_status()


def test_reserve_copies_shared_pages_before_they_are_written(ctx):
    """Four beams of one prompt: the partly filled page is copied for each, the full ones stay shared."""
    import b200attn
    m = Model(np.random.default_rng(0), 4, 4, 12, 16, layers=3, share=0, fill=0)
    m.table[0, :3] = 5, 2, 9
    m.refs[[5, 2, 9]] = 1
    t = m.device()
    b200attn.pages_fork(ctx, t["table"], t["refs"], _dev([0, 0, 0, 0]))
    m.fork(np.zeros(4, np.int32))
    lens, new = np.full(4, 40, np.int32), np.full(4, 10, np.int32)  # positions 40..49: slots 2 and 3
    b200attn.pages_reserve(ctx, t["table"], t["refs"], _dev(lens), _dev(new), t["pages"], 16, t["counts"])
    m.reserve(lens, new)
    m.check(t)
    assert m.counts.tolist() == [8, 0] and m.refs[5] == 4 and m.refs[9] == 0


def test_reserve_all_or_nothing(ctx):
    import b200attn
    m = Model(np.random.default_rng(1), 3, 6, 7, 16, share=0, fill=0)
    t = m.device()
    lens, new = np.zeros(3, np.int32), np.asarray([40, 48, 17], np.int32)  # 3 + 3 + 2 pages, 7 free
    b200attn.pages_reserve(ctx, t["table"], t["refs"], _dev(lens), _dev(new), t["pages"], 16, t["counts"])
    m.reserve(lens, new)
    m.check(t)
    assert m.counts.tolist() == [0, 1]
    new[2] = 16
    b200attn.pages_reserve(ctx, t["table"], t["refs"], _dev(lens), _dev(new), t["pages"], 16, t["counts"])
    m.reserve(lens, new)
    m.check(t)
    assert m.counts.tolist() == [7, 0]


def test_whole_pool_in_use_and_empty_pool(ctx):
    import b200attn
    m = Model(np.random.default_rng(2), 2, 40, 64, 16, share=0, fill=0)
    t = m.device()
    b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"], t["counts"])
    m.compact()
    m.check(t)
    lens, new = np.zeros(2, np.int32), np.full(2, 512, np.int32)
    for _ in range(2):  # all 64 pages; then nothing to do
        b200attn.pages_reserve(ctx, t["table"], t["refs"], _dev(lens), _dev(new), t["pages"], 16, t["counts"])
        m.reserve(lens, new)
        m.check(t)
    b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"], t["counts"])
    m.compact()
    m.check(t)


def test_pages_refusals_and_device_checks(ctx):
    import torch
    import b200attn
    m = Model(np.random.default_rng(3), 3, 4, 12, 16)
    t = m.device()
    z = _dev([0, 0, 0])
    with pytest.raises(ValueError, match="parents"):
        b200attn.pages_fork(ctx, t["table"], t["refs"], z[:2])
    with pytest.raises(ValueError, match="int32"):
        b200attn.pages_fork(ctx, t["table"].long(), t["refs"], z)
    with pytest.raises(ValueError, match="keep_to"):
        b200attn.pages_free(ctx, t["table"], t["refs"], None, None, 16)
    with pytest.raises(ValueError, match="page_size"):
        b200attn.pages_free(ctx, t["table"], t["refs"], None, z, 0)
    with pytest.raises(ValueError, match="pages must be"):
        b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"][:, :5].contiguous(), t["counts"])
    with pytest.raises(ValueError, match="16"):
        b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"][:, :, :15].contiguous(), t["counts"])
    with pytest.raises(ValueError, match="counts"):
        b200attn.pages_reserve(ctx, t["table"], t["refs"], z, z, t["pages"], 16, t["counts"][:1])
    m.check(t)
    b200attn.pages_fork(ctx, t["table"], t["refs"], _dev([0, 9, 2]))  # row 1's entry is refused, others stand
    with pytest.raises(b200attn.B200RuntimeException, match="parents"):
        ctx.check_device_status()
    m.check(t)
    b200attn.pages_reserve(ctx, t["table"], t["refs"], z, _dev([0, 1000, 0]), t["pages"], 16, t["counts"])
    with pytest.raises(b200attn.B200RuntimeException, match="ctx_lens"):
        ctx.check_device_status()
    m.counts[:] = 0
    m.check(t)


def test_graph_replays_of_a_step(ctx):
    """A captured step (trim, fork, reserve, compact) replayed: each replay acts on the state it finds."""
    import torch
    import b200attn
    rng = np.random.default_rng(9)
    m = Model(rng, 12, 10, 200, 16, share=0.2, fill=0.4)
    m.lens = np.minimum(m.lens, 60).astype(np.int32)
    t = m.device()
    new = np.full(12, 9, np.int32)
    parents = np.asarray([0, 0, 2, 3, 1, 5, 6, 6, -1, 9, 10, 11], np.int32)
    new_d, parents_d = _dev(new), _dev(parents)

    def step():
        b200attn.pages_free(ctx, t["table"], t["refs"], None, t["lens"], 16)
        b200attn.pages_fork(ctx, t["table"], t["refs"], parents_d)
        b200attn.pages_reserve(ctx, t["table"], t["refs"], t["lens"], new_d, t["pages"], 16, t["counts"])
        b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"], t["counts"])

    def model_step():
        m.free(None, m.lens)
        m.fork(parents)
        m.reserve(m.lens, new)
        m.compact()

    step()
    model_step()
    m.check(t)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        model_step()
        m.check(t)
    del g
    ctx.check_device_status()


def test_entries_beyond_the_pool_are_reported(ctx):
    """An entry >= num_pages raises the status in every operation that meets it and changes no count.  reserve, free
    and compact leave it; fork hands it on like any other entry and replaces it in a row that gets a parent."""
    import b200attn
    bad = 10 ** 6

    def fresh():
        m = Model(np.random.default_rng(4), 3, 4, 12, 16, share=0, fill=0)
        m.table[0, :2], m.table[1, :2], m.table[2, :1] = (0, 1), (4, bad), (9,)
        m.refs[[0, 1, 4, 9]] = 1
        return m, m.device()

    def reported():
        with pytest.raises(b200attn.B200RuntimeException, match="page_table") as ei:
            ctx.check_device_status()
        assert ei.value.status == b200attn.B2A_EDEVICE
        ctx.check_device_status()

    m, t = fresh()  # row 1 writes positions 20..39: slot 1 is the bad one, slot 2 gets the lowest free page
    b200attn.pages_reserve(ctx, t["table"], t["refs"], _dev([0, 20, 0]), _dev([0, 20, 0]), t["pages"], 16, t["counts"])
    reported()
    m.table[1, 2], m.refs[2] = 2, 1
    m.counts[:] = 1, 0
    m.check(t)
    m, t = fresh()  # the bad slot alone is written: nothing to give out
    b200attn.pages_reserve(ctx, t["table"], t["refs"], _dev([0, 20, 0]), _dev([0, 1, 0]), t["pages"], 16, t["counts"])
    reported()
    m.check(t)
    m, t = fresh()
    b200attn.pages_free(ctx, t["table"], t["refs"], None, _dev([0, 0, 0]), 16)
    reported()
    m.table[:] = -1
    m.table[1, 1] = bad
    m.refs[:] = 0
    m.check(t)
    m, t = fresh()
    b200attn.pages_compact(ctx, t["table"], t["refs"], t["pages"], t["counts"])
    reported()
    m.compact()
    m.check(t)
    for parents in ([0, 0, 2], [0, 1, 1], [0, -1, 2]):
        m, t = fresh()
        b200attn.pages_fork(ctx, t["table"], t["refs"], _dev(parents))
        reported()
        m.table = np.where(np.asarray(parents)[:, None] >= 0, m.table[np.maximum(parents, 0)], -1).astype(np.int32)
        m.refs[:] = 0
        np.add.at(m.refs, m.table[(m.table >= 0) & (m.table < 12)], 1)
        m.check(t)
