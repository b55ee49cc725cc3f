"""Attention over the cache in 4 bits against 64 bits: lengths, heads, types, windows, sinks, absent pages, what lies around the rows."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv4_reference as ref
import lumi_b200

pytestmark = pytest.mark.gpu
PAGE = 64
F32, BF16 = torch.float32, torch.bfloat16


def ok(status):
    lumi_b200.api.check(status)


def work_bytes():
    n = C.c_int64()
    ok(lumi_b200.lib().lumi_k_kv4_attention_work_bytes(16, 1, 256, 256, C.byref(n)))
    return n.value


class Batch:
    """Sequences that hold `held` tokens and bring `new` rows, in a cache of random bytes otherwise (scales that are no numbers among them)."""

    def __init__(self, held, new, heads, kv_heads, dk, dv, dtype=F32, pad=0, seed=0, sharp=1.0, vsize=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.held, self.new, self.heads, self.kv_heads, self.dk, self.dv, self.dtype = list(held), list(new), heads, kv_heads, dk, dv, dtype
        self.total = [a + b for a, b in zip(held, new)]
        self.width = max([1] + [(t + PAGE - 1) // PAGE for t in self.total]) + 1
        self.n_pages = sum((t + PAGE - 1) // PAGE for t in self.total) + 2
        block = ref.block_bytes(dk, dv)
        self.cache = rng.integers(0, 256, (self.n_pages, kv_heads, block), dtype=np.uint8)
        self.cache[:, :, ref.groups(dk) * PAGE * 16:ref.groups(dk) * PAGE * 18] = 0xFF                  # scales of tokens that nobody wrote: NaN
        self.cache[:, :, block - ref.groups(dv) * PAGE * 2:] = 0xFF
        ids, used = rng.permutation(self.n_pages), 0
        self.table = np.full((len(held), self.width), -1, np.int64)
        self.rows = sum(new)
        kv = torch.tensor(self.cache, device="cuda")
        slots = []
        for s, t in enumerate(self.total):
            need = (t + PAGE - 1) // PAGE
            self.table[s, :need] = ids[used:used + need]
            used += need
            slots.append(self.table[s, np.arange(t) // PAGE] * PAGE + np.arange(t) % PAGE)
        self.slots = slots
        every = np.concatenate(slots) if slots else np.zeros(0, np.int64)
        if len(every):
            k = torch.tensor(rng.standard_normal((len(every), kv_heads * dk)), device="cuda", dtype=F32)
            v = torch.tensor(rng.standard_normal((len(every), kv_heads * dv)) * vsize, device="cuda", dtype=F32)
            at = torch.tensor(every, device="cuda", dtype=torch.int32)
            ok(lumi_b200.lib().lumi_k_kv4_append(k.data_ptr(), kv_heads * dk, v.data_ptr(), kv_heads * dv, 0, at.data_ptr(), kv.data_ptr(), self.n_pages, kv_heads, dk, dv, len(every),
                                                 torch.cuda.current_stream().cuda_stream))
        self.kv = kv
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        self.q = torch.full((self.rows + 2, heads * dk + pad), float("nan"), device="cuda", dtype=dtype)
        self.q[:, :heads * dk] = torch.tensor(rng.standard_normal((self.rows + 2, heads * dk)) * sharp, device="cuda").to(dtype)
        self.y = torch.full((self.rows + 2, heads * dv + pad), -5.0, device="cuda", dtype=dtype)
        self.work = torch.zeros(work_bytes(), device="cuda", dtype=torch.uint8)
        self.status = torch.zeros(1, device="cuda", dtype=torch.int32)
        dev = lambda a: torch.tensor(np.asarray(a), device="cuda", dtype=torch.int32)
        self.d_table, self.d_start, self.d_tokens = dev(self.table), dev(self.starts), dev(self.total)
        torch.cuda.synchronize()

    def launch(self, window=0, scale=None, sink=False, max_new=None, rows=None, stream=None, work=None):
        scale = self.dk ** -0.5 if scale is None else scale
        return lumi_b200.lib().lumi_k_kv4_attention(
            self.q.data_ptr(), self.q.stride(0), int(self.dtype == BF16), self.kv.data_ptr(), self.n_pages, self.d_table.data_ptr(), self.width, self.d_start.data_ptr(),
            self.d_tokens.data_ptr(), self.y.data_ptr(), self.y.stride(0), self.heads, self.kv_heads, self.dk, self.dv, window, scale, int(sink), len(self.held),
            self.rows if rows is None else rows, max([0] + self.new) if max_new is None else max_new, (self.work if work is None else work).data_ptr(), self.work.numel(), self.status.data_ptr(),
            torch.cuda.current_stream().cuda_stream if stream is None else stream)

    def sequence(self, s, window=0, scale=None, sink=False):
        """(y, spread) of one sequence in 64 bits."""
        scale = self.dk ** -0.5 if scale is None else scale
        k, v = ref.read(self.kv.cpu().numpy(), self.slots[s], self.dk, self.dv)
        a, b = self.starts[s], self.starts[s + 1]
        q = self.q[a:b, :self.heads * self.dk].double().cpu().numpy().reshape(b - a, self.heads, self.dk)
        return ref.attend(q, k, v, self.held[s], scale, window, sink) + (np.abs(v).max(initial=0.0),)

    def check(self, run=True, status=0, sequences=None, **k):
        if run:
            ok(self.launch(**k))
        torch.cuda.synchronize()
        assert int(self.status) == status
        for s in range(len(self.held)) if sequences is None else sequences:
            y, spread, vmax = self.sequence(s, **{n: v for n, v in k.items() if n in ("window", "scale", "sink")})
            got = self.y[self.starts[s]:self.starts[s + 1], :self.heads * self.dv].double().cpu().numpy().reshape(y.shape)
            # scores: two fp16 terms of q and up to 32 sums in fp32, 2^-18 of sum |q k|; softmax weights as two fp16 terms (fp32 rows) or one (bf16 rows, 2^-11); one rounding of y
            slack = vmax * (spread[..., None] * 2.0 ** -18 + (2.0 ** -11 if self.dtype == BF16 else 2.0 ** -18))
            tol = slack + np.abs(y) * (2.0 ** -8 if self.dtype == BF16 else 2.0 ** -24)
            assert np.isfinite(got).all() and (np.abs(got - y) <= tol).all(), (s, np.abs(got - y).max(), tol.min())
        assert (self.y[self.rows:] == -5.0).all() and (self.y[:, self.heads * self.dv:] == -5.0).all()      # rows behind the last, columns behind the heads


TYPES = [F32, BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("held", [0, 1, 62, 63, 64, 127, 300, 1000, 5000])
def test_one_token_of_one_sequence(held, dtype):
    Batch([held], [1], 4, 2, 64, 64, dtype, seed=held).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dk,dv", [(1, 1, 1, 1), (2, 2, 32, 32), (3, 1, 33, 40), (4, 4, 48, 64), (8, 2, 64, 128), (5, 1, 80, 80), (12, 3, 96, 96), (8, 1, 100, 60),
                                                 (16, 2, 128, 128), (20, 2, 128, 64), (16, 1, 160, 160), (24, 1, 192, 128), (16, 1, 256, 256), (40, 2, 64, 256), (2, 1, 256, 1)])
def test_heads(heads, kv_heads, dk, dv, dtype):
    Batch([70, 0, 200], [1, 1, 1], heads, kv_heads, dk, dv, dtype, pad=3, seed=dk).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("held,new", [([3, 700, 64, 0], [1, 1, 1, 1]), ([3, 700, 64, 0], [2, 1, 4, 3]), ([10, 100, 0, 63], [0, 5, 0, 1]), ([0, 0], [0, 0]), ([130, 1], [17, 64]), ([0, 5, 200], [65, 128, 1]),
                                      ([0], [300]), ([77], [200]), ([1000, 64], [33, 100])])
def test_rows_of_several_tokens(held, new, dtype):
    Batch(held, new, 8, 2, 64, 64, dtype, seed=len(held)).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dk,dv", [(4, 4, 128, 128), (6, 2, 80, 40), (1, 1, 256, 256), (32, 2, 48, 96), (3, 3, 33, 1), (7, 1, 128, 64)])
def test_prompts_of_other_heads(heads, kv_heads, dk, dv, dtype):
    Batch([0, 40, 129], [70, 1, 90], heads, kv_heads, dk, dv, dtype, seed=dk, pad=1).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 100000])
def test_windows_and_sinks(window, sink, dtype):
    Batch([500, 3, 64, 150], [1, 1, 1, 1], 4, 2, 64, 64, dtype, seed=window).check(window=window, sink=sink)
    Batch([500, 3, 64, 150], [3, 70, 0, 130], 4, 2, 64, 64, dtype, seed=window).check(window=window, sink=sink)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_key_inside_and_outside_the_window(dtype):
    """The value of one far token is planted: it counts for the last row that sees it, and not for the next."""
    for new in (1, 90):
        b = Batch([400], [new], 2, 1, 64, 64, dtype, seed=9)
        y0, _, _ = b.sequence(0, window=100)
        spot = 400 - 100 + (new > 1)                                     # seen by row 0 (by rows 0 and 1 of many)
        for at, seen in ((spot, new > 1), (spot + 1, True)):
            v = torch.full((1, 64), 1000.0, device="cuda")
            slot = torch.tensor([b.slots[0][at]], device="cuda", dtype=torch.int32)
            k = torch.zeros(1, 64, device="cuda")
            ok(lumi_b200.lib().lumi_k_kv4_append(k.data_ptr(), 64, v.data_ptr(), 64, 0, slot.data_ptr(), b.kv.data_ptr(), b.n_pages, 1, 64, 64, 1, torch.cuda.current_stream().cuda_stream))
            b.check(window=100)
            assert (float(b.y[0, :64].float().abs().max()) > 1.0) == seen or new > 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30])
def test_scales_of_scores(scale, dtype):
    Batch([200, 10], [1, 40], 4, 2, 64, 64, dtype).check(scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("qsize,vsize", [(1e-20, 1.0), (1e3, 1.0), (1.0, 1e-25), (1.0, 1e6), (1.0, 1e30), (0.0, 1.0)])
def test_numbers_of_any_size(qsize, vsize, dtype):
    b = Batch([300, 20], [1, 30], 4, 2, 64, 64, dtype, sharp=qsize, vsize=vsize)
    b.check(scale=0.125 if qsize < 100 else 0.125 / qsize)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 70])
def test_values_whose_size_changes_from_page_to_page(new, dtype):
    """Scales grow and shrink by powers of ten along the context; each row is as good as its largest values allow."""
    for order in (1, -1):
        b = Batch([640], [new], 2, 1, 64, 64, dtype, seed=3)
        size = 10.0 ** (order * (np.arange(b.total[0]) // 64 - 5.0))
        rng = np.random.default_rng(4)
        v = torch.tensor(rng.standard_normal((b.total[0], 64)) * size[:, None], device="cuda", dtype=F32)
        k = torch.tensor(rng.standard_normal((b.total[0], 64)), device="cuda", dtype=F32)
        at = torch.tensor(b.slots[0], device="cuda", dtype=torch.int32)
        ok(lumi_b200.lib().lumi_k_kv4_append(k.data_ptr(), 64, v.data_ptr(), 64, 0, at.data_ptr(), b.kv.data_ptr(), b.n_pages, 1, 64, 64, b.total[0], torch.cuda.current_stream().cuda_stream))
        b.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_that_are_no_numbers(dtype):
    """A NaN in the keys of one token and head makes the rows that see it NaN, of that head alone; behind the window it is not looked at."""
    for new in (1, 80):
        b = Batch([200], [new], 2, 2, 64, 64, dtype)
        k, v = torch.zeros(1, 128, device="cuda"), torch.zeros(1, 128, device="cuda")
        k[0, 5] = float("nan")
        at = torch.tensor([b.slots[0][100]], device="cuda", dtype=torch.int32)
        ok(lumi_b200.lib().lumi_k_kv4_append(k.data_ptr(), 128, v.data_ptr(), 128, 0, at.data_ptr(), b.kv.data_ptr(), b.n_pages, 2, 64, 64, 1, torch.cuda.current_stream().cuda_stream))
        ok(b.launch())
        torch.cuda.synchronize()
        assert torch.isnan(b.y[:new, :64]).all() and torch.isfinite(b.y[:new, 64:128]).all()
        b.y.fill_(-5.0)
        b.check(window=100)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,new", [(1, 1), (4, 1), (2, 3), (1, 12), (8, 4), (1, 90), (4, 40)])
def test_values_that_are_no_numbers(group, new, dtype):
    """A NaN or an infinity in the values of a token and head makes the rows that see the token NaN, of that head alone; the other rows of the same call are as without it."""
    window, held, d = 100, 300, 64
    for spot in (held - window - 5, held - window, held - window + new // 2, held - 3, held + new // 2):
        b = Batch([held, 70], [new, 1], 2 * group, 2, d, d, dtype, seed=spot)
        v = torch.ones(1, 2 * d, device="cuda")
        v[0, 3] = float("nan") if spot % 2 else float("inf")
        at = torch.tensor([b.slots[0][spot]], device="cuda", dtype=torch.int32)
        k = torch.zeros(1, 2 * d, device="cuda")
        put = lambda: ok(lumi_b200.lib().lumi_k_kv4_append(k.data_ptr(), 2 * d, v.data_ptr(), 2 * d, 0, at.data_ptr(), b.kv.data_ptr(), b.n_pages, 2, d, d, 1, torch.cuda.current_stream().cuda_stream))
        put()
        ok(b.launch(window=window))
        torch.cuda.synchronize()
        got = b.y[:b.rows, :2 * group * d].clone().view(b.rows, 2, group * d)
        v.fill_(1.0)                                                     # (the same token with numbers)
        put()
        b.check(window=window)
        whole = b.y[:b.rows, :2 * group * d].view(b.rows, 2, group * d)
        for row in range(b.rows):
            sees = row < new and held + row - window < spot <= held + row
            assert torch.isnan(got[row, 0]).all() if sees else torch.isfinite(got[row, 0]).all()
            close = lambda x, y: (x.float() - y.float()).abs().max() <= 2.0 ** (-6 if dtype == BF16 else -14)
            assert close(got[row, 1], whole[row, 1]) and (sees or close(got[row, 0], whole[row, 0]))


@pytest.mark.parametrize("held,new,heads,d", [(31, 1, 16, 64), (4000, 1, 16, 64), (4000, 2, 4, 128), (1000, 1, 32, 256), (9000, 1, 4, 80), (1000, 40, 16, 64), (300, 300, 8, 128)])
def test_fp32_rows_keep_their_precision(held, new, heads, d):
    """The whole result's error: two fp16 terms of q and of weights (2^-22 each), scores of up to 2^4 in units of log2 in fp32 (2^-20), exponentials (2^-21), and sums of up to 2^5 products of the
    tensor cores, which cut off (2^-19 of a score or a result): 2^-18 of the result, whose numbers are sums that cancel about as much as the errors do."""
    b = Batch([held], [new], heads, 4, d, d, F32, seed=held + new)
    b.check()
    want = b.sequence(0)[0]
    got = b.y[:new, :heads * d].double().cpu().numpy().reshape(want.shape)
    assert np.linalg.norm(got - want) <= 2.0 ** -18 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_that_are_no_numbers(dtype):
    for new in (1, 70):
        b = Batch([100], [new], 2, 1, 64, 64, dtype)
        b.q[0, 3] = float("nan")
        ok(b.launch())
        torch.cuda.synchronize()
        assert torch.isnan(b.y[0, :64]).all() and torch.isfinite(b.y[0, 64:128]).all() and torch.isfinite(b.y[1:new, :128]).all()


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_not_there(dtype, sink):
    """Tokens of a page that is none of the cache's are passed over, and a row that sees nothing else is zero."""
    for new in (1, 70):
        b = Batch([200, 20], [new, new], 2, 1, 64, 64, dtype)
        table = b.table.copy()
        table[0, 1], table[1, :] = b.n_pages, -1
        b.d_table = torch.tensor(table, device="cuda", dtype=torch.int32)
        ok(b.launch(sink=sink))
        torch.cuda.synchronize()
        assert int(b.status) == 1
        keep = np.r_[0:64, 128:b.total[0]]
        k, v = ref.read(b.kv.cpu().numpy(), b.slots[0][keep], 64, 64)
        got = b.y[:b.rows, :128].double().cpu().numpy().reshape(b.rows, 2, 64)
        for i in range(new):
            q = b.q[i:i + 1, :128].double().cpu().numpy().reshape(1, 2, 64)
            n = 200 + i + 1 - 64
            want, _ = ref.attend(q, k[:n], v[:n], n - 1, 0.125, 0, sink)
            assert np.abs(got[i] - want[0]).max() <= 2.0 ** -6 if dtype == BF16 else 2.0 ** -14
        assert (got[new:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_that_do_not_fit(dtype):
    """Rows of a sequence whose lengths make no sense are left as they were; the others are computed."""
    b = Batch([100, 50, 10, 5], [1, 2, 1, 1], 2, 1, 64, 64, dtype)
    for tokens, start in (([101, 52, 10 ** 6, 6], b.starts), ([101, 1, 11, 6], b.starts), ([101, 52, -5, 6], b.starts), ([101, 52, 11, 6], [0, 1, 3, 4, 50])):
        b.status.zero_()
        b.y.fill_(-5.0)
        b.d_tokens = torch.tensor(tokens, device="cuda", dtype=torch.int32)
        b.d_start = torch.tensor(np.asarray(start), device="cuda", dtype=torch.int32)
        left = [s for s in range(4) if tokens[s] != b.total[s] or start[s + 1] != b.starts[s + 1]]
        b.check(status=1, sequences=[s for s in range(4) if s not in left], max_new=2)
        for s in left:
            assert (b.y[b.starts[s]:b.starts[s + 1]] == -5.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_beyond_max_new_are_left_out(dtype):
    b = Batch([100, 50], [3, 1], 2, 1, 64, 64, dtype)
    ok(b.launch(max_new=1))
    torch.cuda.synchronize()
    assert (b.y[:3] == -5.0).all()
    b.check(run=False, sequences=[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences(dtype):
    rng = np.random.default_rng(7)
    held, new = rng.integers(0, 400, 700), rng.integers(0, 3, 700)
    b = Batch(held, new, 4, 2, 32, 32, dtype)
    b.check(sequences=range(0, 700, 23))
    assert not (b.y[:b.rows] == -5.0).all(1).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_call_gives_the_same_bits(dtype):
    b = Batch([3000, 100, 7000], [1, 1, 1], 8, 2, 128, 128, dtype)
    b.check()
    first = b.y.clone()
    for _ in range(5):
        b.y.fill_(-5.0)
        ok(b.launch())
        torch.cuda.synchronize()
        assert torch.equal(first, b.y)


@pytest.mark.parametrize("new", [1, 100])
def test_captured_and_replayed_over_growing_contexts(new):
    """Lengths lie on the device: a captured call follows them."""
    b = Batch([900, 500], [new, 1], 8, 2, 64, 64, BF16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ok(b.launch(stream=side.cuda_stream))
    full = list(b.held)
    for cut in (0, 1, 64, 333, 450):
        b.held = [h - cut for h in full]
        b.total = [h + n for h, n in zip(b.held, b.new)]
        b.slots = [s[:t] for s, t in zip(b.slots, b.total)]
        b.d_tokens.copy_(torch.tensor(b.total, dtype=torch.int32))
        b.y.fill_(-5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        b.check(run=False)


def test_two_calls_at_once_on_two_streams():
    bs = [Batch([4000, 900], [1, 50], 8, 2, 64, 64, BF16, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    for _ in range(10):
        for b, s in zip(bs, streams):
            ok(b.launch(stream=s.cuda_stream))
    torch.cuda.synchronize()
    for b in bs:
        b.check(run=False)


def test_far_slots():
    """Pages whose bytes lie beyond 2^31 of the cache's beginning."""
    b = Batch([200], [1], 2, 2, 128, 128, BF16)
    block = ref.block_bytes(128, 128)
    n_pages = (1 << 31) // (2 * block) + 5000
    far = torch.zeros(n_pages * 2 * block, device="cuda", dtype=torch.uint8).view(n_pages, 2, block)
    shift = n_pages - b.n_pages
    far[shift:] = b.kv
    b.kv, b.n_pages = far, n_pages
    b.d_table = torch.tensor(np.where(b.table >= 0, b.table + shift, -1), device="cuda", dtype=torch.int32)
    ok(b.launch())
    b.kv, b.n_pages = far[shift:].clone(), n_pages - shift
    b.check(run=False)


def test_a_step_as_it_is_used():
    """Plan, norm, append and attention of three steps, captured as one graph, against the reference: a prompt first, then single tokens."""
    rng = np.random.default_rng(11)
    heads, kv_heads, d, width, n_pages, nseq, lib = 8, 2, 64, 4, 16, 3, lumi_b200.lib()
    i32 = lambda a: torch.tensor(np.asarray(a), device="cuda", dtype=torch.int32)
    page = C.c_int64()
    ok(lib.lumi_k_kv4_page_bytes(kv_heads, d, d, C.byref(page)))
    kv = torch.full((n_pages, page.value), 0xFF, device="cuda", dtype=torch.uint8)
    tokens, new = i32([0] * nseq), i32([0] * nseq)
    table, free, pool = i32(np.full((nseq, width), -1)), i32(rng.permutation(n_pages)), i32([n_pages, 0])
    rows = 160
    start, pos, slot = i32([0] * (nseq + 1)), i32([0] * rows), i32([0] * rows)
    width_x = heads * d
    x, o = torch.zeros(rows, width_x, device="cuda"), torch.zeros(rows, width_x, device="cuda", dtype=BF16)
    y, ones = torch.zeros(rows, width_x, device="cuda", dtype=BF16), torch.ones(width_x, device="cuda")
    q, out = y, torch.zeros(rows, width_x, device="cuda", dtype=BF16)
    k, v = torch.zeros(rows, kv_heads * d, device="cuda", dtype=BF16), torch.zeros(rows, kv_heads * d, device="cuda", dtype=BF16)
    work, status = torch.zeros(work_bytes(), device="cuda", dtype=torch.uint8), i32([0])

    def step(st):
        ok(lib.lumi_k_page_plan(tokens.data_ptr(), new.data_ptr(), nseq, table.data_ptr(), width, free.data_ptr(), n_pages, pool.data_ptr(), pool.data_ptr(), tokens.data_ptr(),
                                start.data_ptr(), pos.data_ptr(), slot.data_ptr(), rows, st))
        ok(lib.lumi_k_block_norm(x.data_ptr(), 0, width_x, o.data_ptr(), 1, width_x, ones.data_ptr(), 0, 0, 1.0, ones.data_ptr(), y.data_ptr(), 1, width_x, rows, width_x, 1e-5, st))
        ok(lib.lumi_k_kv4_append(k.data_ptr(), kv_heads * d, v.data_ptr(), kv_heads * d, 1, slot.data_ptr(), kv.data_ptr(), n_pages, kv_heads, d, d, rows, st))
        ok(lib.lumi_k_kv4_attention(q.data_ptr(), width_x, 1, kv.data_ptr(), n_pages, table.data_ptr(), width, start.data_ptr(), tokens.data_ptr(), out.data_ptr(), width_x, heads, kv_heads,
                                    d, d, 0, 0.125, 0, nseq, rows, 100, work.data_ptr(), work.numel(), status.data_ptr(), st))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(side.cuda_stream)
    held = [[np.zeros((0, kv_heads, d)), np.zeros((0, kv_heads, d))] for _ in range(nseq)]
    for lens in ([100, 3, 0], [1, 1, 50], [1, 1, 1], [-1, 1, 1], [70, 1, 1]):
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        for t in (x, o, k, v):
            t.copy_(torch.tensor(rng.standard_normal(t.shape), device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(status) == 0 and int(pool[1]) == 0
        at = 0
        for s, n in enumerate(lens):
            if n < 0:
                held[s] = [np.zeros((0, kv_heads, d)), np.zeros((0, kv_heads, d))]
            n = max(n, 0)
            if n == 0:
                continue
            for i, t in enumerate((k, v)):
                fresh = t[at:at + n].float().cpu().numpy().reshape(n, kv_heads, d)
                held[s][i] = np.concatenate([held[s][i], ref.values(*ref.quantise(fresh))])
            qs = q[at:at + n].double().cpu().numpy().reshape(n, heads, d)
            want, spread = ref.attend(qs, held[s][0], held[s][1], len(held[s][0]) - n, 0.125, 0, False)
            got = out[at:at + n].double().cpu().numpy().reshape(want.shape)
            tol = np.abs(held[s][1]).max() * (spread[..., None] * 2.0 ** -18 + 2.0 ** -11) + np.abs(want) * 2.0 ** -8
            assert (np.abs(got - want) <= tol).all()
            at += n
        assert at == int(start[-1])
