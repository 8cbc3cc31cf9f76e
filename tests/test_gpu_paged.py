"""The paged KV-cache operators on the GPU against their definitions in 64 bits.

Tolerances follow from the arithmetic, with u = 2^-24 (half an ulp of f32
relative to the value) and e = finfo(t).eps / 2 for a 16-bit type t:
  rotation   one rounding e |y|, cos and sin within 2^-21 of |x0| + |x1|
  scores     d = 2 u (head_dim + 4) max_j scale sum |q k| each (a matrix unit may
             cut rather than round, hence 2 u a step), and 4 u |x| for scaling
  out        the probabilities' rounding e, twice the scores' error (numerator
             and sum), 2^-20 for exp and the sums, all on sum p |v|; the final
             rounding e |out|; for f16 probabilities below the normal range
             2^-25 sum |v| relative to the row's largest, and outputs 2^-25
  lse        the scores' error, 2^-20 and n u for the sum of n terms
  mass       per key, (2 d + 2^-20 (1 + |lse|)) of its sum and rows u of it
Evictions are exact.
"""
from __future__ import annotations

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def P():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for the gpu tests")
    from jetsonfabric_b200 import paged
    return paged


def rand(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)


class Case:
    """A pool, a page table in no order, and ragged sequences. Everything that
    must not be read holds NaN: other pages, slots behind the keys, rows behind
    the last sequence."""

    def __init__(self, P, new, kv, kv_heads=2, hd=128, page_size=16, dtype=torch.float16, seed=0, pad=0, heads_first=False, extra=0,
                 fill=True):
        self.P, self.new, self.kv, self.ps, self.kvh, self.hd, self.dtype = P, new, kv, page_size, kv_heads, hd, dtype
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        host = torch.Generator().manual_seed(seed)
        n = len(kv)
        self.width = max(1, max((-(-k // page_size) for k in kv), default=1)) + extra
        pages = n * self.width + 2
        shape = (pages, kv_heads, page_size, hd) if heads_first else (pages, page_size, kv_heads, hd)
        self.k_pool, self.v_pool = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        if heads_first:
            self.k_pool, self.v_pool = self.k_pool.transpose(1, 2), self.v_pool.transpose(1, 2)
        self.table_host = torch.randperm(pages, generator=host)[:n * self.width].view(n, self.width)
        self.table = self.table_host.to(torch.int32).cuda()
        self.keys = [rand(g, k, kv_heads, hd, dtype=dtype) for k in kv]
        self.values = [rand(g, k, kv_heads, hd, dtype=dtype) for k in kv]
        if fill:
            for b in range(n):
                self.put(b, 0, self.keys[b], self.values[b])
        starts = [0]
        for c in new:
            starts.append(starts[-1] + c)
        self.starts, self.rows = starts, starts[-1] + pad
        self.q_start = torch.tensor(starts, dtype=torch.int32).cuda()
        self.kv_len = torch.tensor(kv, dtype=torch.int32).cuda()
        self.cache = P.PagedCache(self.k_pool, self.v_pool)
        self.batch = P.PagedBatch(self.q_start, self.kv_len, self.table)
        self.error = torch.zeros(1, dtype=torch.int32, device="cuda")

    def where(self, b, slots):
        return self.table_host[b, slots // self.ps].cuda(), (slots % self.ps).cuda()

    def put(self, b, at, k, v):
        page, place = self.where(b, torch.arange(at, at + k.shape[0]))
        self.k_pool[page, place] = k
        self.v_pool[page, place] = v

    def queries(self, heads, std=1.5):
        q = torch.full((self.rows, heads, self.hd), math.nan, dtype=self.dtype, device="cuda")
        n = self.starts[-1]
        q[:n] = rand(self.g, n, heads, self.hd, dtype=self.dtype, std=std)
        return q


def definition(case, q, scale, window, keys=None, values=None):
    """Per sequence: scores x and their error bound d [heads, rows, keys], the mask."""
    keys, values = keys or case.keys, values or case.values
    for b, (n, kv) in enumerate(zip(case.new, case.kv)):
        r = slice(case.starts[b], case.starts[b + 1])
        G = q.shape[1] // case.kvh
        k = keys[b].double().repeat_interleave(G, 1).permute(1, 0, 2)
        v = values[b].double().repeat_interleave(G, 1).permute(1, 0, 2)
        qd = q[r].double().permute(1, 0, 2)
        x = qd @ k.mT * scale
        pos = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")
        seen = key <= pos
        if window:
            seen = seen & (key > pos - window)
        size = (qd.abs() @ k.abs().mT * scale).masked_fill(~seen, 0)
        d = 2 * U * (case.hd + 4) * size + 4 * U * x.abs()
        yield b, r, x.masked_fill(~seen, -math.inf), d.masked_fill(~seen, 0), v


def check_attention(case, q, out, lse, scale, window, dtype=None, **kw):
    e = torch.finfo(out.dtype).eps / 2
    for b, r, x, d, v in definition(case, q, scale, window, **kw):
        if x.shape[1] == 0:
            continue
        got, got_lse = out[r].double().permute(1, 0, 2), lse[r].double().T
        if x.shape[2] == 0:
            assert torch.all(got == 0) and torch.all(got_lse == -math.inf)
            continue
        want_lse = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(want_lse.isinf(), 0.0, want_lse)[..., None])
        want = p @ v
        dmax = d.amax(-1)
        n = (x > -math.inf).sum(-1)
        spread = p @ v.abs()
        tol = e * want.abs() + spread * (e + 2 * dmax + 2.0 ** -20 + n * U)[..., None] * 1.01
        if out.dtype == torch.float16:
            top = torch.exp(x.amax(-1) - want_lse).nan_to_num()
            tol = tol + 2.0 ** -25 * (1 + top[..., None] * ((x > -math.inf).double() @ v.abs()))
        assert torch.all((got - want).abs() <= tol), (b, ((got - want).abs() - tol).max())
        empty = want_lse.isinf()
        assert torch.all(got_lse[empty] == -math.inf) and torch.all(got[empty] == 0)
        err = (got_lse - want_lse)[~empty].abs()
        assert torch.all(err <= (dmax + 2.0 ** -20 * (1 + want_lse.abs()) + n * U)[~empty]), (b, err.max())


def run_attention(P, case, q, window=0, scale=None, workspace=None, out=None, **kw):
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full((case.rows, q.shape[1]), 7.0, device="cuda")
    P.attention(q, case.cache, case.batch, out, P.attention_workspace() if workspace is None else workspace, scale=scale,
                window=window, lse=lse, error_flag=case.error, **kw)
    torch.cuda.synchronize()
    n = case.starts[-1]
    assert torch.all(out[n:] == 7.0) and torch.all(lse[n:] == 7.0)  # rows of no sequence
    return out, lse


SHAPES = [
    # new, kv, heads, kv_heads, head_dim, page_size, window, pad
    ([1], [1], 2, 2, 128, 16, 0, 0),
    ([1], [777], 12, 2, 128, 16, 0, 0),
    ([1, 1, 1], [1, 128, 129], 28, 4, 128, 16, 0, 1),
    ([1] * 5, [5, 2000, 64, 1, 513], 14, 2, 64, 32, 0, 0),
    ([1, 0, 1, 2], [300, 40, 17, 2], 16, 2, 128, 64, 0, 2),
    ([1, 1], [4000, 900], 6, 1, 128, 8, 300, 0),
    ([1], [5000], 40, 1, 128, 128, 0, 0),          # 40 query heads share one kv head
    ([3, 17, 1], [3, 100, 260], 28, 4, 128, 16, 0, 3),
    ([33, 5], [700, 5], 8, 8, 96, 16, 0, 0),
    ([100], [100], 12, 2, 64, 1024, 17, 0),
    ([1, 9], [40, 300], 4, 2, 24, 16, 0, 0),        # head_dim below one swizzled row
    ([40, 130], [1500, 131], 28, 4, 128, 16, 0, 1),
    ([257, 64, 1], [257, 1000, 1], 16, 2, 128, 256, 0, 0),
    ([300], [1300], 40, 8, 128, 16, 200, 2),
    ([129, 7, 250], [2000, 900, 300], 5, 1, 64, 64, 0, 5),
    ([512], [513], 2, 2, 104, 32, 0, 0),
    ([1000], [1000], 7, 1, 128, 128, 1, 0),         # a window of one: every row sees itself
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,kv,heads,kv_heads,hd,ps,window,pad", SHAPES)
def test_attention(P, dtype, new, kv, heads, kv_heads, hd, ps, window, pad):
    case = Case(P, new, kv, kv_heads, hd, ps, dtype, seed=len(new) + hd, pad=pad, heads_first=len(kv) % 2 == 1)
    q = case.queries(heads)
    scale = hd ** -0.5
    workspace = P.attention_workspace()
    out, lse = run_attention(P, case, q, window, workspace=workspace)
    check_attention(case, q, out, lse, scale, window)
    again, lse2 = run_attention(P, case, q, window, workspace=workspace)
    assert torch.equal(out.nan_to_num(), again.nan_to_num()) and torch.equal(lse, lse2)  # bit for bit
    assert int(case.error) == 0


@pytest.mark.parametrize("new,kv", [([3, 1], [0, 0]), ([5, 2], [2, 1]), ([200], [60]), ([400, 3], [100, 0])])
def test_rows_before_the_first_slot_see_nothing(P, new, kv):
    """More new rows than keys: the first rows lie before slot 0."""
    case = Case(P, new, kv, extra=1)
    q = case.queries(8)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)
    assert int(case.error) == 0


@pytest.mark.parametrize("new", [1, 200])
def test_large_scores_and_constant_rows(P, new):
    """Scores in the hundreds (one key takes all the weight) and rows whose scores are all equal."""
    case = Case(P, [new, new], [600, 601], dtype=torch.bfloat16)
    q = case.queries(8, std=60.0)
    q[new // 2] = 0
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)


@pytest.mark.parametrize("new", [1, 150])
def test_growing_maximum(P, new):
    """Every later key scores higher: the running maximum grows in each tile."""
    case = Case(P, [new], [2000], kv_heads=1, dtype=torch.float16, fill=False)
    direction = rand(case.g, 128)
    direction /= direction.norm()
    ramp = torch.linspace(-30, 30, 2000, device="cuda")[:, None, None]
    case.keys = [(direction * ramp).half().reshape(2000, 1, 128)]
    case.put(0, 0, case.keys[0], case.values[0])
    q = case.queries(6)
    q[:] = (direction * 40).half()
    out, lse = run_attention(P, case, q, scale=0.1)
    check_attention(case, q, out, lse, 0.1, 0)


@pytest.mark.parametrize("new", [1, 180])
def test_rows_at_strides(P, new):
    """q a slice of a fused projection, out a slice of a wider buffer, both untouched elsewhere."""
    case = Case(P, [new, new], [300, 555], pad=1)
    heads = 12
    fused = torch.full((case.rows, (heads + 4) * 128), 3.0, dtype=case.dtype, device="cuda")
    q = fused[:, :heads * 128]
    q.copy_(case.queries(heads).nan_to_num().reshape(case.rows, -1))
    wide = torch.full((case.rows, 2 + heads, 128), 7.0, dtype=case.dtype, device="cuda")
    out, lse = run_attention(P, case, q.unflatten(1, (heads, 128)), out=wide[:, 1:1 + heads])
    check_attention(case, q.unflatten(1, (heads, 128)), out, lse, 128 ** -0.5, 0)
    assert torch.all(wide[:, 0] == 7.0) and torch.all(wide[:, -1] == 7.0) and torch.all(fused[:, heads * 128:] == 3.0)


@pytest.mark.parametrize("new", [1, 140])
def test_bad_pages_read_as_zeros_and_are_flagged(P, new):
    case = Case(P, [new, new], [400, 400])
    case.table[0, 3] = -5
    case.table[1, 20] = case.k_pool.shape[0]
    case.table[1, 24] = 2 ** 31 - 1
    for b, page in ((0, 3), (1, 20), (1, 24)):
        case.keys[b][page * 16:page * 16 + 16] = 0
        case.values[b][page * 16:page * 16 + 16] = 0
    q = case.queries(8)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)
    assert int(case.error) == P.ERROR_RANGE


def test_bad_lengths_are_cut_and_flagged(P):
    """A length beyond the table counts as the table's keys; a row range outside the rows as none."""
    case = Case(P, [1, 1], [64, 64])
    case.kv_len[0] = 10 ** 9
    q = case.queries(4)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)
    assert int(case.error) == P.ERROR_RANGE
    case.error.zero_()
    case.kv_len[0] = 64
    case.q_start[2] = 50
    out, lse = run_attention(P, case, q)
    assert torch.all(out[1] == 7.0) and int(case.error) == P.ERROR_RANGE
    case.kv_len[1] = -3
    case.q_start[2] = 2
    out, lse = run_attention(P, case, q)
    assert torch.all(out[1] == 0) and torch.all(lse[1] == -math.inf)


@pytest.mark.parametrize("new,heads,window", [(1, 4, 300), (40, 4, 300), (1000, 8, 24)])
def test_slots_near_the_largest(P, new, heads, window):
    """A context of 2^31 - 1024 keys whose table repeats one page, seen through a window; more is cut."""
    case = Case(P, [new], [1024], kv_heads=1, page_size=1024)
    table = case.table.expand(1, 1 << 21).contiguous()
    kv_len = torch.tensor([2 ** 31 - 1], dtype=torch.int32).cuda()
    case.batch = P.PagedBatch(case.q_start, kv_len, table)
    q = case.queries(heads)
    out, lse = run_attention(P, case, q, window)
    assert int(case.error) == P.ERROR_RANGE
    check_attention(case, q, out, lse, 128 ** -0.5, window)  # the last slots are the page's last
    kv_len.fill_(2 ** 31 - 1024)
    again, lse2 = run_attention(P, case, q, window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    k = rand(case.g, new, 1, 128)
    pos = torch.arange(new, dtype=torch.int32, device="cuda")
    P.rope_append(q, k.half(), k.half(), pos, P.Rope(torch.zeros(64, dtype=torch.float64, device="cuda")), case.cache, case.batch,
                  torch.empty_like(q))
    torch.cuda.synchronize()
    page, place = case.where(0, torch.arange(1024 - new, 1024))
    assert torch.equal(case.k_pool[page, place], k.half())


@pytest.mark.parametrize("new,kv,heads,kvh,hd", [([9], [200], 132, 1, 64), ([40, 1], [90, 300], 300, 2, 128), ([64], [64], 128, 1, 128)])
def test_large_groups(P, new, kv, heads, kvh, hd):
    """More query heads per kv head than a tile has rows, and exactly as many."""
    case = Case(P, new, kv, kvh, hd)
    q = case.queries(heads)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, hd ** -0.5, 0)
    before = torch.rand(len(kv), kvh, max(kv), device="cuda", generator=case.g)
    got = torch.empty_like(before)
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before, error_flag=case.error)
    torch.cuda.synchronize()
    check_mass(case, q, lse, before, got, hd ** -0.5, 0)
    assert int(case.error) == 0


@pytest.mark.parametrize("new", [1, 50])
def test_a_pool_of_one_page_shared_by_sequences(P, new):
    case = Case(P, [new, 0, new], [60, 64, 64], kv_heads=1, hd=64, page_size=64)
    pool = case.k_pool[:1].clone()
    pool[0] = rand(case.g, 64, 1, 64, dtype=case.dtype)
    case.cache = P.PagedCache(pool, pool)
    case.batch = P.PagedBatch(case.q_start, case.kv_len, torch.zeros(3, 1, dtype=torch.int32, device="cuda"))
    case.keys = case.values = [pool[0, :k] for k in case.kv]
    q = case.queries(8)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 0.125, 0)
    assert int(case.error) == 0


@pytest.mark.parametrize("new", [1, 100])
def test_masses_shorter_than_the_keys(P, new):
    """Only the slots that have a mass get one, and the cut is flagged."""
    case = Case(P, [new, new], [400, 150])
    q = case.queries(8)
    out, lse = run_attention(P, case, q)
    before = torch.rand(2, 2, 170, device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before, error_flag=case.error)
    wide = torch.full((2, 2, 400), 9.0, device="cuda")
    wide[:, :, :170] = before
    full = torch.full_like(wide, 9.0)
    P.attention_mass(q, lse, case.cache, case.batch, full, mass_in=wide)
    torch.cuda.synchronize()
    assert int(case.error) == P.ERROR_RANGE
    check_mass(case, q, lse, wide, full, 128 ** -0.5, 0)
    # the same positive terms, new x 4 heads and `before`, in an order that the items' cut may
    # change: each sum of n of them is off by at most n U of itself
    assert torch.allclose(got, full[:, :, :170], rtol=2 * (4 * new + 8) * U, atol=0)
    assert torch.all(got[1, :, 150:] == 9.0)


@pytest.mark.parametrize("new,kv,heads", [([1] * 3, [900, 20, 400], 16), ([200, 90], [700, 90], 16)])
def test_captured_calls_follow_new_lengths(P, new, kv, heads):
    """One captured attention replayed after the lengths and the pages changed, next to a second
    captured one with its own workspace, and on another stream than the inputs'."""
    case = Case(P, new, kv, extra=30)
    q = case.queries(heads)
    workspaces = [P.attention_workspace() for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in range(2)]
    lses = [torch.zeros(case.rows, heads, device="cuda") for _ in range(2)]
    run_attention(P, case, q)
    graphs = []
    for ws, out, lse in zip(workspaces, outs, lses):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            P.attention(q, case.cache, case.batch, out, ws, lse=lse)
            P.attention(q, case.cache, case.batch, out, ws, lse=lse)
        graphs.append(graph)
    for step in range(3):
        case.kv = [k + 37 * step for k in kv]
        case.kv_len.copy_(torch.tensor(case.kv, dtype=torch.int32))
        case.keys = [rand(case.g, k, case.kvh, case.hd, dtype=case.dtype) for k in case.kv]
        case.values = [rand(case.g, k, case.kvh, case.hd, dtype=case.dtype) for k in case.kv]
        for b in range(len(kv)):
            case.put(b, 0, case.keys[b], case.values[b])
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for out, lse in zip(outs, lses):
            check_attention(case, q, out, lse, 128 ** -0.5, 0)


def test_calls_on_two_streams_and_devices(P):
    case = Case(P, [1, 70], [500, 200])
    q = case.queries(8)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    out, lse = run_attention(P, case, q, stream=side)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)
    if torch.cuda.device_count() > 1:
        with torch.cuda.device(1):
            out, lse = run_attention(P, case, q, workspace=P.attention_workspace("cuda:0"))
            torch.cuda.synchronize(0)
        check_attention(case, q, out, lse, 128 ** -0.5, 0)


def test_offsets_beyond_32_bits(P):
    """Pages at the end of a pool of more than 2^32 elements."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough device memory")
    ps, kvh, hd = 1024, 8, 128
    pages = (1 << 32) // (ps * kvh * hd) + 3
    pool = torch.empty(pages, ps, kvh, hd, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    kv = 1500
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32).cuda()
    q_start, kv_len = torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.tensor([kv], dtype=torch.int32).cuda()
    cache, batch = P.PagedCache(pool, pool), P.PagedBatch(q_start, kv_len, table)
    keys = rand(g, kv, kvh, hd, dtype=torch.float16)
    pool[pages - 1] = keys[:ps]
    pool[pages - 3, :kv - ps] = keys[ps:]
    q = rand(g, 2, 16, hd)
    zero = torch.zeros(64, dtype=torch.float64, device="cuda")
    # angles of zero: the append stores k and v as they are (v last, the pools are one)
    q16 = torch.empty(2, 16, hd, dtype=torch.float16, device="cuda")
    kn = rand(g, 2, kvh, hd)
    P.rope_append(q, kn, kn, torch.zeros(2, dtype=torch.int32, device="cuda"), P.Rope(zero), cache, batch, q16)
    keys[-2:] = kn.half()
    out, lse = torch.empty_like(q16), torch.empty(2, 16, device="cuda")
    P.attention(q16, cache, batch, out, P.attention_workspace(), lse=lse)
    torch.cuda.synchronize()
    assert torch.equal(q16, q.half())
    case = Case.__new__(Case)
    case.new, case.kv, case.starts, case.kvh, case.hd = [2], [kv], [0, 2], kvh, hd
    case.keys = case.values = [keys]
    check_attention(case, q16, out, lse, hd ** -0.5, 0)
    # compaction to the front of the same far pages
    mass = torch.rand(1, kvh, kv, device="cuda", generator=g)
    keep = torch.empty(1, kvh, 100, dtype=torch.int32, device="cuda")
    P.evict(mass, cache, batch, keep, kv_len, recent=10)
    torch.cuda.synchronize()
    for h in range(kvh):
        assert torch.equal(pool[pages - 1, :100, h], keys[keep[0, h].long(), h])
    assert int(kv_len) == 100


# ---- rotation and append ------------------------------------------------------------

def rotated(x, pos, freq, factor, interleaved):
    """(rotated x in 64 bits, the bound on |x0| + |x1| of each element)."""
    x = x.double()
    dims = 2 * freq.numel()
    angle = pos.double()[:, None, None] * freq
    cos, sin = torch.cos(angle) * factor, torch.sin(angle) * factor
    part, rest = x[..., :dims], x[..., dims:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        size = torch.stack((a.abs() + b.abs(),) * 2, -1).flatten(-2)
    else:
        a, b = part.chunk(2, -1)
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        size = torch.cat((a.abs() + b.abs(),) * 2, -1)
    return torch.cat((y, rest), -1), torch.cat((size * factor, torch.zeros_like(rest)), -1)


def close(got, want, size):
    e = torch.finfo(got.dtype).eps / 2
    least = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    return torch.all((got.double() - want).abs() <= e * want.abs() + (1 + e) * 2.0 ** -21 * size + least)


@pytest.mark.parametrize("source,dtype", [(torch.float32, torch.float16), (torch.float32, torch.bfloat16), (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("heads,kv_heads,hd,dims,interleaved", [
    (12, 2, 128, 128, False), (28, 4, 128, 128, True), (4, 2, 64, 64, False), (5, 1, 96, 48, False), (6, 3, 128, 72, True),
    (3, 1, 40, 6, False), (2, 2, 24, 2, True), (7, 1, 128, 66, False), (4, 4, 8, 8, False)])
def test_rope_append(P, source, dtype, heads, kv_heads, hd, dims, interleaved):
    new, kv = [1, 0, 17, 3], [5, 9, 17, 300]
    case = Case(P, new, kv, kv_heads, hd, 16, dtype, seed=dims, pad=2, heads_first=interleaved)
    g = case.g
    q, k, v = (rand(g, case.rows, h, hd, dtype=source) for h in (heads, kv_heads, kv_heads))
    q_out = torch.full((case.rows, heads, hd), 7.0, dtype=dtype, device="cuda")
    pos = torch.randint(-5, 1 << 20, (case.rows,), dtype=torch.int32, device="cuda", generator=g)
    rope = P.Rope.scaled(dims, 1e6, "yarn", interleaved=interleaved, factor=4.0, trained=32768) if dims > 2 else \
        P.Rope.scaled(dims, 1e6, interleaved=interleaved)
    before_k, before_v = case.k_pool.clone(), case.v_pool.clone()
    P.rope_append(q, k, v, pos, rope, case.cache, case.batch, q_out, error_flag=case.error)
    torch.cuda.synchronize()
    n = case.starts[-1]
    factor = rope.desc.factor
    assert close(q_out[:n], *rotated(q[:n], pos[:n], rope.freq, factor, interleaved))
    assert torch.all(q_out[n:] == 7.0)
    want, size = rotated(k[:n], pos[:n], rope.freq, factor, interleaved)
    for b in range(len(new)):
        r = slice(case.starts[b], case.starts[b + 1])
        page, place = case.where(b, torch.arange(kv[b] - new[b], kv[b]))
        assert close(case.k_pool[page, place], want[r], size[r])
        assert torch.equal(case.v_pool[page, place], v[r].to(dtype))
        case.k_pool[page, place] = before_k[page, place]
        case.v_pool[page, place] = before_v[page, place]
    # nothing else was touched (NaNs compare by their bits)
    assert torch.equal(case.k_pool.view(torch.int16), before_k.view(torch.int16))
    assert torch.equal(case.v_pool.view(torch.int16), before_v.view(torch.int16))
    assert int(case.error) == 0


@pytest.mark.parametrize("rows", [1, 5, 5000])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_fused_rows_in_place(P, rows, interleaved):
    """q, k and v are slices of one projection whose rows are 4 elements off 16 bytes, then of an aligned one
    rotated in place."""
    heads, kvh, hd = 6, 2, 64
    for odd in (4, 0):
        case = Case(P, [rows], [rows + 3], kvh, hd, 32, torch.bfloat16, seed=rows)
        fused = rand(case.g, rows, (heads + 2 * kvh) * hd + odd, dtype=torch.bfloat16)
        q, k, v = fused[:, :heads * hd], fused[:, heads * hd:(heads + kvh) * hd], fused[:, (heads + kvh) * hd:(heads + 2 * kvh) * hd]
        pos = torch.arange(rows, dtype=torch.int32, device="cuda")
        rope = P.Rope.scaled(hd, 1e4, interleaved=interleaved)
        want_q, size_q = rotated(q.unflatten(1, (heads, hd)), pos, rope.freq, 1.0, interleaved)
        want_k, size_k = rotated(k.unflatten(1, (kvh, hd)), pos, rope.freq, 1.0, interleaved)
        v_was = v.clone()
        q_out = q if odd == 0 else torch.empty(rows, heads * hd, dtype=torch.bfloat16, device="cuda")
        P.rope_append(q, k, v, pos, rope, case.cache, case.batch, q_out)
        torch.cuda.synchronize()
        assert close(q_out.unflatten(1, (heads, hd)), want_q, size_q)
        page, place = case.where(0, torch.arange(3, rows + 3))
        assert close(case.k_pool[page, place], want_k, size_k)
        assert torch.equal(case.v_pool[page, place], v_was.unflatten(1, (kvh, hd)))


def test_rope_skips_bad_slots(P):
    case = Case(P, [3, 1], [2, 40], extra=1)
    case.table[1, 2] = 10 ** 6
    before = case.k_pool.clone()
    q, k = rand(case.g, 4, 4, 128), rand(case.g, 4, 2, 128)
    out = torch.zeros(4, 4, 128, dtype=torch.float16, device="cuda")
    rope = P.Rope(torch.zeros(64, dtype=torch.float64, device="cuda"))
    P.rope_append(q, k, k, torch.zeros(4, dtype=torch.int32, device="cuda"), rope, case.cache, case.batch, out, error_flag=case.error)
    torch.cuda.synchronize()
    assert torch.equal(out, q.half()) and int(case.error) == P.ERROR_RANGE
    page, place = case.where(0, torch.arange(2))
    assert torch.equal(case.k_pool[page, place], k[1:3].half())  # row 0 lies before slot 0
    case.k_pool[page, place] = before[page, place]
    assert torch.equal(case.k_pool.view(torch.int16), before.view(torch.int16))


def test_rope_appends_nothing_beyond_the_table(P):
    """A length beyond the table: the row that has no slot must not take the last one's."""
    case = Case(P, [2, 1], [64, 64])
    case.kv_len[0] = 65  # new tokens at slots 63 and 64, the table holds 64
    case.kv_len[1] = 2 ** 31 - 1
    before = case.k_pool.clone()
    q, k = rand(case.g, 3, 4, 128), rand(case.g, 3, 2, 128)
    out = torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    rope = P.Rope(torch.zeros(64, dtype=torch.float64, device="cuda"))
    P.rope_append(q, k, k, torch.zeros(3, dtype=torch.int32, device="cuda"), rope, case.cache, case.batch, out, error_flag=case.error)
    torch.cuda.synchronize()
    assert torch.equal(out, q.half()) and int(case.error) == P.ERROR_RANGE
    page, place = case.where(0, torch.arange(63, 64))
    assert torch.equal(case.k_pool[page, place], k[:1].half())
    case.k_pool[page, place] = before[page, place]
    assert torch.equal(case.k_pool.view(torch.int16), before.view(torch.int16))


# ---- accumulated weight ----------------------------------------------------------------

def check_mass(case, q, lse, before, got, scale, window):
    for b, r, x, d, v in definition(case, q, scale, window):
        n, kv = case.new[b], case.kv[b]
        seen = x > -math.inf
        l = lse[r].double().T[..., None]
        p = torch.where(seen, torch.exp(x - torch.where(seen, l, 0.0)), 0.0)
        err = p * (2 * d + 2.0 ** -20 * (1 + x.abs().masked_fill(~seen, 0) + torch.where(seen, l.abs(), 0.0)))
        G = q.shape[1] // case.kvh
        added = p.unflatten(0, (case.kvh, G)).sum((1, 2))
        tol = err.unflatten(0, (case.kvh, G)).sum((1, 2)) + added * U * (n * G + 8)
        old = torch.zeros_like(added) if before is None else before[b, :, :kv].double()
        old[:, max(0, kv - n):] = 0
        want = old + added
        assert torch.all((got[b, :, :kv].double() - want).abs() <= tol + 2 * U * want), b


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,kv,heads,kv_heads,hd,ps,window,pad", SHAPES)
def test_mass(P, dtype, new, kv, heads, kv_heads, hd, ps, window, pad):
    case = Case(P, new, kv, kv_heads, hd, ps, dtype, seed=3 * len(new) + hd, pad=pad, heads_first=len(kv) % 2 == 0)
    q = case.queries(heads)
    out, lse = run_attention(P, case, q, window)
    slots = max(kv) + 5
    before = torch.rand(len(kv), kv_heads, slots, device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before, window=window, error_flag=case.error)
    torch.cuda.synchronize()
    check_mass(case, q, lse, before, got, hd ** -0.5, window)
    for b, k in enumerate(kv):
        assert torch.all(got[b, :, k:] == 9.0)  # slots behind the keys
    # in place, and again from nothing: bit for bit what the first call gave
    twice = before.clone()
    P.attention_mass(q, lse, case.cache, case.batch, twice, mass_in=twice, window=window)
    fresh = torch.full_like(before, math.nan)
    P.attention_mass(q, lse, case.cache, case.batch, fresh, window=window)
    torch.cuda.synchronize()
    for b, k in enumerate(kv):
        assert torch.equal(twice[b, :, :k], got[b, :, :k]) and torch.equal(twice[b, :, k:], before[b, :, k:])
    check_mass(case, q, lse, None, fresh, hd ** -0.5, window)
    assert int(case.error) == 0


def test_mass_of_a_sequence_without_new_rows(P):
    case = Case(P, [0, 2], [50, 1], extra=1)
    q = case.queries(4)
    lse = torch.full((2, 4), -math.inf, device="cuda")
    lse[1] = 0.0
    before = torch.rand(2, 2, 60, device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    q.zero_()
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before)
    torch.cuda.synchronize()
    assert torch.equal(got[0, :, :50], before[0, :, :50]) and torch.all(got[0, :, 50:] == 9.0)
    # the row before slot 0 (lse = -inf) sees nothing; the other gives e^0 from each of 2 heads
    assert torch.all(got[1, :, 0] == 2.0)


# ---- eviction -----------------------------------------------------------------------------

def kept_slots(weights, n, budget, recent):
    if n <= budget:
        return list(range(n))
    early = sorted(range(n - recent), key=lambda j: (-(weights[j] if weights[j] == weights[j] else -math.inf), weights[j] != weights[j], j))
    return sorted(early[:budget - recent] + list(range(n - recent, n)))


def test_empty_batches(P):
    """No new rows: only the masses go over. No sequences: nothing happens."""
    case = Case(P, [0, 0], [50, 200])
    flag, ws = case.error, P.attention_workspace()
    empty = torch.empty(0, 4, 128, dtype=torch.float16, device="cuda")
    kv = torch.empty(0, 2, 128, dtype=torch.float16, device="cuda")
    lse, pos = torch.empty(0, 4, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    rope = P.Rope(torch.ones(64, dtype=torch.float64, device="cuda"))
    before = torch.rand(2, 2, 210, device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    nobody = P.PagedBatch(case.q_start[:1], case.kv_len[:0], case.table[:0])
    for batch, x, y in ((case.batch, before, got), (nobody, before[:0], got[:0])):
        P.rope_append(empty, kv, kv, pos, rope, case.cache, batch, empty, error_flag=flag)
        P.attention(empty, case.cache, batch, empty, ws, lse=lse, error_flag=flag)
        P.attention_mass(empty, lse, case.cache, batch, y, mass_in=x, error_flag=flag)
    P.evict(before[:0], case.cache, nobody, torch.empty(0, 2, 16, dtype=torch.int32, device="cuda"), case.kv_len[:0], recent=0)
    torch.cuda.synchronize()
    for b, k in enumerate(case.kv):
        assert torch.equal(got[b, :, :k], before[b, :, :k]) and torch.all(got[b, :, k:] == 9.0)
    assert int(flag) == 0


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kv,budget,recent,kv_heads,hd,ps", [
    ([1], 1, 0, 2, 128, 16), ([700], 512, 64, 2, 128, 16), ([5, 300, 64, 65, 0], 64, 10, 4, 128, 8), ([200, 90], 33, 33, 1, 96, 32),
    ([100, 1000], 99, 0, 3, 64, 16), ([2500, 513, 512, 511], 512, 1, 2, 128, 64), ([9000], 2000, 500, 1, 24, 1024),
    ([40] * 40, 16, 4, 8, 128, 16)])
def test_evict(P, in_place, kv, budget, recent, kv_heads, hd, ps):
    n = len(kv)
    case = Case(P, [0] * n, kv, kv_heads, hd, ps, torch.bfloat16, seed=budget, heads_first=n % 2 == 0, extra=-(-budget // ps))
    slots = max(kv) + 3
    mass = torch.rand(n, kv_heads, slots, device="cuda", generator=case.g).pow(-2) - 1
    # many ties: only a few values, zeros of both signs among them
    ties = torch.randint(0, 6, mass.shape, device="cuda", generator=case.g)
    mass = torch.where(ties == 0, 0.0, torch.where(ties == 1, -0.0, torch.where(ties == 2, 1.25, mass)))
    if slots > 50:
        mass[0, 0, 7] = math.nan
        mass[0, 0, 11] = math.inf
    mass[:, :, max(kv):] = math.inf  # behind every key
    weights = mass.cpu().tolist()
    keep = torch.full((n, kv_heads, budget), 99, dtype=torch.int32, device="cuda")
    length = case.kv_len if in_place else torch.empty_like(case.kv_len)
    if in_place:
        table, mass_out = case.table_host, mass
        P.evict(mass, case.cache, case.batch, keep, length, recent=recent, error_flag=case.error)
    else:
        wide = max(max(-(-k // ps) for k in kv), 0)
        # the spare columns of the table are pages that no key uses
        new_table = case.table[:, wide:].contiguous()
        table, mass_out = case.table_host[:, wide:], torch.full((n, kv_heads, budget), 9.0, device="cuda")
        P.evict(mass, case.cache, case.batch, keep, length, recent=recent, mass_out=mass_out, page_table_out=new_table,
                error_flag=case.error)
    torch.cuda.synchronize()
    assert length.tolist() == [min(k, budget) for k in kv] and int(case.error) == 0
    for b, k in enumerate(kv):
        m = min(k, budget)
        slot = torch.arange(m)
        page, place = table[b, slot // ps].cuda(), (slot % ps).cuda()
        for h in range(kv_heads):
            want = kept_slots(weights[b][h], k, budget, recent)
            assert keep[b, h].tolist() == want + [-1] * (budget - m), (b, h)
            at = torch.tensor(want, dtype=torch.long).cuda()
            assert torch.equal(case.k_pool[page, place, h], case.keys[b][at, h])
            assert torch.equal(case.v_pool[page, place, h], case.values[b][at, h])
            old = torch.tensor(weights[b][h], device="cuda")[at]
            assert torch.equal(mass_out[b, h, :m].nan_to_num(-5.0), old.nan_to_num(-5.0))
    if not in_place:  # the old pages stay as they were
        for b in range(n):
            page, place = case.where(b, torch.arange(kv[b]))
            assert torch.equal(case.k_pool[page, place], case.keys[b])


def test_evict_flags_bad_pages(P):
    case = Case(P, [0], [100], extra=2)
    mass = torch.arange(200, 0, -1, device="cuda", dtype=torch.float32).expand(1, 2, 200).contiguous()
    case.table[0, 1] = -1
    before = case.k_pool.clone()
    keep = torch.empty(1, 2, 32, dtype=torch.int32, device="cuda")
    P.evict(mass, case.cache, case.batch, keep, torch.empty_like(case.kv_len), recent=0, mass_out=torch.empty_like(keep, dtype=torch.float32),
            page_table_out=case.table[:, 7:9].contiguous(), error_flag=case.error)
    torch.cuda.synchronize()
    assert int(case.error) == P.ERROR_RANGE
    assert torch.equal(keep[0, 0], torch.arange(32, dtype=torch.int32, device="cuda"))
    spare = case.table_host[0, 7:9]
    assert torch.equal(case.k_pool[spare[0]], case.keys[0][:16])
    assert torch.equal(case.k_pool[spare[1]].view(torch.int16), before[spare[1]].view(torch.int16))  # not moved


@pytest.mark.parametrize("hd", [128, 24])
def test_evict_refuses_a_copy_of_the_table(P, hd):
    """Out of place within a sequence's own pages: nothing is moved, and the call says so."""
    case = Case(P, [0, 0], [3000, 40], hd=hd)
    mass = torch.rand(2, 2, 3000, device="cuda", generator=case.g)
    before_k, before_v = case.k_pool.clone(), case.v_pool.clone()
    keep = torch.empty(2, 2, 1000, dtype=torch.int32, device="cuda")
    P.evict(mass, case.cache, case.batch, keep, torch.empty_like(case.kv_len), recent=10, mass_out=torch.empty(2, 2, 1000, device="cuda"),
            page_table_out=case.table.clone(), error_flag=case.error)
    torch.cuda.synchronize()
    assert int(case.error) == P.ERROR_RANGE
    assert torch.equal(case.k_pool.view(torch.int16), before_k.view(torch.int16))
    assert torch.equal(case.v_pool.view(torch.int16), before_v.view(torch.int16))


def test_evict_leaves_uncut_sequences_on_their_pages(P):
    """A sequence within the budget may keep its pages while another moves to new ones."""
    case = Case(P, [0, 0], [300, 40], extra=7)
    mass = torch.rand(2, 2, 300, device="cuda", generator=case.g)
    weights = mass.cpu().tolist()
    table = case.table[:, :7].clone()
    table[0] = case.table[0, 19:26]
    keep, length = torch.empty(2, 2, 100, dtype=torch.int32, device="cuda"), torch.empty_like(case.kv_len)
    P.evict(mass, case.cache, case.batch, keep, length, recent=10, mass_out=torch.empty(2, 2, 100, device="cuda"),
            page_table_out=table, error_flag=case.error)
    torch.cuda.synchronize()
    assert int(case.error) == 0 and length.tolist() == [100, 40]
    for b, h in ((0, 0), (0, 1), (1, 0), (1, 1)):
        want = torch.tensor(kept_slots(weights[b][h], case.kv[b], 100, 10)).cuda()
        slot = torch.arange(len(want), device="cuda")
        assert torch.equal(case.k_pool[table[b, slot // 16].long(), slot % 16, h], case.keys[b][want, h])
        assert torch.equal(case.v_pool[table[b, slot // 16].long(), slot % 16, h], case.values[b][want, h])


@pytest.mark.parametrize("kv,budget", [(500, 1100000), (1100000, 1060000)])
def test_evict_with_a_budget_beyond_the_grid(P, kv, budget):
    """Out of place, a budget of more steps than a grid has rows: of a short sequence, and of one that fills it."""
    g = torch.Generator(device="cuda").manual_seed(budget)
    ps, hd, room = 1024, 128, 136  # rows of 16-byte pieces that are not whole 32-byte sectors
    old, new = -(-kv // ps), -(-min(kv, budget) // ps)
    store = torch.empty(2, old + new, ps, 1, room, dtype=torch.float16, device="cuda")
    for pool in store:
        for page in pool:
            page.copy_(torch.randn(page.shape, device="cuda", generator=g))
    k_pool, v_pool = store[0, ..., :hd], store[1, ..., :hd]
    table = torch.randperm(old + new, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    width = -(-budget // ps)
    new_table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")  # pages that nothing is kept in are not read
    new_table[0, :new] = table[old:]
    kv_len = torch.tensor([kv], dtype=torch.int32, device="cuda")
    cache = P.PagedCache(k_pool, v_pool)
    batch = P.PagedBatch(torch.zeros(2, dtype=torch.int32, device="cuda"), kv_len, table[None, :old].contiguous())
    mass = torch.randint(0, 1000, (1, 1, kv), device="cuda", generator=g).float()
    keep = torch.empty(1, 1, budget, dtype=torch.int32, device="cuda")
    length, mass_out = torch.empty_like(kv_len), torch.zeros(1, 1, budget, device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    P.evict(mass, cache, batch, keep, length, recent=100, mass_out=mass_out, page_table_out=new_table, error_flag=error)
    torch.cuda.synchronize()
    kept = min(kv, budget)
    assert int(length) == kept and int(error) == 0
    if kv > budget:
        early = torch.sort(mass[0, 0, :kv - 100], descending=True, stable=True).indices[:budget - 100]
        want = torch.cat((torch.sort(early).values, torch.arange(kv - 100, kv, device="cuda")))
    else:
        want = torch.arange(kv, device="cuda")
    assert torch.equal(keep[0, 0, :kept].long(), want) and torch.all(keep[0, 0, kept:] == -1)
    assert torch.equal(mass_out[0, 0, :kept], mass[0, 0, want])
    at = torch.arange(kept, device="cuda")
    for pool in (k_pool, v_pool):
        source = pool[table[want // ps].long(), want % ps, 0]
        assert torch.equal(pool[new_table[0, at // ps].long(), at % ps, 0], source)


# ---- as they are used together ----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_conversation_through_all_of_them(P, dtype):
    """Prompt chunks, decode steps, an eviction in place and more decode, captured where the calls
    repeat, against a cache kept in 64-bit lists."""
    heads, kvh, hd, ps, budget, recent = 12, 2, 128, 16, 96, 24
    n, width = 3, 20
    g = torch.Generator(device="cuda").manual_seed(5)
    pool = torch.zeros(n * width, ps, kvh, hd, dtype=dtype, device="cuda")
    k_pool, v_pool = pool, pool.clone()
    table = torch.randperm(n * width, generator=torch.Generator().manual_seed(1)).view(n, width).to(torch.int32).cuda()
    rope = P.Rope.scaled(hd, 1e6, "yarn", factor=4.0, trained=64)
    cache = P.PagedCache(k_pool, v_pool)
    workspace = P.attention_workspace()
    kv_len = torch.zeros(n, dtype=torch.int32, device="cuda")
    mass = torch.full((n, kvh, width * ps), math.nan, device="cuda")
    keys = [torch.empty(0, kvh, hd, dtype=dtype, device="cuda") for _ in range(n)]
    values = list(keys)
    position = [0] * n

    def step(new):
        starts = [0]
        for c in new:
            starts.append(starts[-1] + c)
        rows = starts[-1]
        q_start = torch.tensor(starts, dtype=torch.int32).cuda()
        kv_len.add_(q_start[1:] - q_start[:-1])
        batch = P.PagedBatch(q_start, kv_len, table)
        q, k, v = (rand(g, rows, h, hd) for h in (heads, kvh, kvh))
        pos = torch.tensor([position[b] + i for b in range(n) for i in range(new[b])], dtype=torch.int32).cuda()
        q16, out = (torch.empty(rows, heads, hd, dtype=dtype, device="cuda") for _ in range(2))
        lse = torch.empty(rows, heads, device="cuda")
        before = mass.clone()
        P.rope_append(q, k, v, pos, rope, cache, batch, q16)
        P.attention(q16, cache, batch, out, workspace, lse=lse)
        P.attention_mass(q16, lse, cache, batch, mass, mass_in=mass)
        torch.cuda.synchronize()
        want_k, size = rotated(k, pos, rope.freq, rope.desc.factor, False)
        case = Case.__new__(Case)
        case.kvh, case.hd, case.new, case.starts, case.kv = kvh, hd, new, starts, kv_len.tolist()
        for b in range(n):
            r = slice(starts[b], starts[b + 1])
            slot = torch.arange(case.kv[b] - new[b], case.kv[b])
            page, place = table[b, (slot // ps).cuda()].long(), (slot % ps).cuda()
            assert close(k_pool[page, place], want_k[r], size[r])
            keys[b] = torch.cat((keys[b], k_pool[page, place]))
            values[b] = torch.cat((values[b], v[r].to(dtype)))
            position[b] += new[b]
        case.keys, case.values = keys, values
        check_attention(case, q16, out, lse, hd ** -0.5, 0)
        check_mass(case, q16, lse, before, mass, hd ** -0.5, 0)

    step([70, 0, 33])
    step([50, 129, 1])
    for _ in range(3):
        step([1, 1, 1])
    batch = P.PagedBatch(torch.zeros(n + 1, dtype=torch.int32, device="cuda"), kv_len, table)
    keep = torch.empty(n, kvh, budget, dtype=torch.int32, device="cuda")
    lengths, weights = kv_len.tolist(), mass.cpu().tolist()
    P.evict(mass, cache, batch, keep, kv_len, recent=recent)
    torch.cuda.synchronize()
    assert kv_len.tolist() == [min(k, budget) for k in lengths]
    for b in range(n):
        for h in range(kvh):
            assert keep[b, h][:min(lengths[b], budget)].tolist() == kept_slots(weights[b][h], lengths[b], budget, recent)
        at = keep[b, :, :min(lengths[b], budget)].long().T
        keys[b] = torch.stack([keys[b][at[:, h], h] for h in range(kvh)], 1)
        values[b] = torch.stack([values[b][at[:, h], h] for h in range(kvh)], 1)
    step([1, 1, 1])
    step([17, 1, 40])


# ---- the whole range, at random ---------------------------------------------------------------

@pytest.mark.parametrize("seed", range(40))
def test_random_batches(P, seed):
    """Random shapes through attention and accumulated weight, twice with one workspace: right and bit for bit the same."""
    import random
    rng = random.Random(seed)
    kv_heads = rng.choice([1, 2, 3, 8])
    group = rng.choice([1, 2, 3, 5, 6, 7, 8, 16, 24])
    hd = rng.choice([8, 64, 72, 128, 128])
    ps = rng.choice([8, 16, 64, 256])
    window = rng.choice([0, 0, 1, 7, 130, 1000])
    n = rng.choice([1, 2, 5, 40, 150])
    most = max(2, 6000 // n)
    kv = [rng.choice([0, 1, rng.randrange(1, most), rng.randrange(1, most)]) for _ in range(n)]
    longest = rng.choice([1, 1, 4, 40, 300])
    new = [min(k + rng.choice([0, 0, 0, 2]), rng.choice([0, 1, rng.randrange(1, longest + 1)])) for k in kv]
    if sum(new) == 0:
        new[0], kv[0] = 1, max(1, kv[0])
    dtype = rng.choice([torch.float16, torch.bfloat16])
    case = Case(P, new, kv, kv_heads, hd, ps, dtype, seed=seed, pad=rng.randrange(3), heads_first=rng.random() < 0.5)
    q = case.queries(kv_heads * group)
    workspace = P.attention_workspace()
    out, lse = run_attention(P, case, q, window, workspace=workspace)
    check_attention(case, q, out, lse, hd ** -0.5, window)
    again, lse2 = run_attention(P, case, q, window, workspace=workspace)
    assert torch.equal(out.nan_to_num(), again.nan_to_num()) and torch.equal(lse, lse2)
    mass = torch.full((n, kv_heads, max(max(kv), 1)), math.nan, device="cuda")
    P.attention_mass(q, lse, case.cache, case.batch, mass, window=window, error_flag=case.error)
    torch.cuda.synchronize()
    check_mass(case, q, lse, None, mass, hd ** -0.5, window)
    assert int(case.error) == 0


@pytest.mark.parametrize("n", [129, 700, 4096])
@pytest.mark.parametrize("new", [1, 7])
def test_many_sequences(P, n, new):
    """More sequences than a warp's registers hold, up to the most a call takes."""
    kv = [new + (b * 37) % 90 for b in range(n)]
    case = Case(P, [new] * n, kv, 1, 64, 16, torch.bfloat16, seed=n)
    q = case.queries(8)
    out, lse = run_attention(P, case, q)
    mass = torch.full((n, 1, max(kv)), math.nan, device="cuda")
    P.attention_mass(q, lse, case.cache, case.batch, mass)
    torch.cuda.synchronize()
    for b in range(0, n, max(1, n // 60)):  # each sequence like a case of its own
        one = Case.__new__(Case)
        one.new, one.kv, one.kvh, one.hd = [new], [kv[b]], 1, 64
        one.starts, one.keys, one.values = [0, new], [case.keys[b]], [case.values[b]]
        r = slice(case.starts[b], case.starts[b + 1])
        check_attention(one, q[r], out[r], lse[r], 0.125, 0)
        check_mass(one, q[r], lse[r], None, mass[b:b + 1], 0.125, 0)


def test_one_long_context_over_all_ctas(P):
    """One sequence of 60000 keys, split over every CTA and joined, for a single token and for a chunk."""
    for new in (1, 20, 300):
        case = Case(P, [new], [60000], 2, 128, 64, torch.float16, seed=new)
        q = case.queries(4)
        workspace = P.attention_workspace()
        out, lse = run_attention(P, case, q, workspace=workspace)
        check_attention(case, q, out, lse, 128 ** -0.5, 0)
        for _ in range(5):
            again, lse2 = run_attention(P, case, q, workspace=workspace)
            assert torch.equal(out, again) and torch.equal(lse, lse2)
        mass = torch.empty(1, 2, 60000, device="cuda")
        P.attention_mass(q, lse, case.cache, case.batch, mass)
        torch.cuda.synchronize()
        check_mass(case, q, lse, None, mass, 128 ** -0.5, 0)


def test_evict_beyond_the_selections_cache(P):
    """More keys than the selection holds in registers and in shared memory, in place, with many ties."""
    for kv in ([16385, 70000], [49153, 40000]):
        case = Case(P, [0, 0], kv, 1, 8, 128, torch.float16, seed=kv[0])
        mass = torch.randint(0, 50, (2, 1, max(kv)), device="cuda", generator=case.g).float()
        weights = mass.cpu().tolist()
        keep = torch.empty(2, 1, 20000, dtype=torch.int32, device="cuda")
        P.evict(mass, case.cache, case.batch, keep, case.kv_len, recent=100, error_flag=case.error)
        torch.cuda.synchronize()
        assert int(case.error) == 0
        for b, k in enumerate(kv):
            m = min(k, 20000)
            want = kept_slots(weights[b][0], k, 20000, 100)
            assert keep[b, 0, :m].tolist() == want and torch.all(keep[b, 0, m:] == -1)
            at = torch.tensor(want).cuda()
            page, place = case.where(b, torch.arange(m))
            assert torch.equal(case.k_pool[page, place], case.keys[b][at])
            assert torch.equal(mass[b, 0, :m], torch.tensor(weights[b][0], device="cuda")[at])


@pytest.mark.parametrize("seqs,new,lo,hi,heads,kvh,window", [
    (150, 20, 100, 400, 8, 2, 0), (150, 30, 40, 300, 6, 1, 50),  # more sequences than a warp's registers hold
    (64, 12, 200, 700, 28, 4, 0), (30, 40, 300, 310, 16, 2, 0),   # many short items
    (4, 200, 1000, 1000, 28, 4, 0), (5, 260, 2000, 2001, 10, 2, 128)])  # few of one length
def test_batches_of_short_chunks(P, seqs, new, lo, hi, heads, kvh, window):
    """Items that are divided whole, in attention and in the accumulated weights."""
    host = torch.Generator().manual_seed(seqs + new)
    kv = torch.randint(lo, hi + 1, (seqs,), generator=host).tolist()
    case = Case(P, [new - b % 3 for b in range(seqs)], kv, kvh, 128, 32, torch.bfloat16, seed=seqs)
    q = case.queries(heads)
    out, lse = run_attention(P, case, q, window)
    check_attention(case, q, out, lse, 128 ** -0.5, window)
    before = torch.rand(seqs, kvh, max(kv), device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before, window=window, error_flag=case.error)
    again = before.clone()
    P.attention_mass(q, lse, case.cache, case.batch, again, mass_in=again, window=window)
    torch.cuda.synchronize()
    check_mass(case, q, lse, before, got, 128 ** -0.5, window)
    for b, k in enumerate(kv):
        assert torch.equal(again[b, :, :k], got[b, :, :k]) and torch.all(got[b, :, k:] == 9.0)
    assert int(case.error) == 0


def test_weak_keys_beside_a_strong_one_count(P):
    """f16 caches: the first key outweighs each of 100,000 others by 2^25.2 and holds zeros, so that the result is
    theirs alone. They must not fall out of the second product: the bound has 2^-32 of the row's largest for what
    f16 cannot hold, where check_attention has 2^-25."""
    strong, n = 17.46875, 100000  # 25.2 ln 2, exact in f16; the others score 0
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for hd, seqs, new, heads in ((128, sms, 1, 8), (64, sms, 1, 8), (128, 1, 4736, 8), (64, 1, 4736, 8)):
        # single tokens over one shared prefix, a sequence per SM; a long chunk over it
        keys = n + new
        width = -(-keys // 128)
        k_pool, v_pool = (torch.zeros(width, 128, 1, hd, dtype=torch.float16, device="cuda") for _ in range(2))
        g = torch.Generator(device="cuda").manual_seed(hd + new)
        value = (torch.rand(hd, device="cuda", generator=g) + 0.5).half()
        v_pool[:] = value
        k_pool[0, 0, 0, 0], v_pool[0, 0] = strong, 0
        q = torch.zeros(seqs * new, heads, hd, dtype=torch.float16, device="cuda")
        q[:, :, 0] = 1.0
        table = torch.arange(width, dtype=torch.int32, device="cuda").expand(seqs, width).contiguous()
        q_start = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device="cuda")
        kv_len = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
        cache, batch = P.PagedCache(k_pool, v_pool), P.PagedBatch(q_start, kv_len, table)
        out, lse = torch.empty_like(q), torch.empty(seqs * new, heads, device="cuda")
        P.attention(q, cache, batch, out, P.attention_workspace(), scale=1.0, lse=lse)
        torch.cuda.synchronize()
        weak = (keys - new + torch.arange(new, device="cuda", dtype=torch.float64)).repeat(seqs)[:, None, None]
        total = math.exp(strong) + weak
        spread = weak / total * value.double()
        e, d = 2.0 ** -11, 2 * U * (hd + 4) * strong + 4 * U * strong
        tol = e * spread + spread * (e + 2 * d + 2.0 ** -20 + weak * U) * 1.01
        tol = tol + 2.0 ** -25 + 2.0 ** -32 * math.exp(strong) / total * weak * value.double()
        err = (out.double() - spread).abs()
        assert torch.all(err <= tol), (hd, new, (err / tol).max())
        want = torch.log(total).squeeze(-1)
        assert torch.all((lse.double() - want).abs() <= d + 2.0 ** -20 * (1 + want) + weak.squeeze(-1) * U)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 700])
def test_scores_near_the_largest_meant(P, new, dtype):
    """Scores up to 2^25, where a step of f32 is 4: the largest takes all the weight, and no exponential leaves its
    type. Neighbouring scores differ by 2^-10 or more of the largest, their error is below 2^-15."""
    case = Case(P, [new], [3000], kv_heads=1, dtype=dtype, fill=False)
    steps = 256 if dtype == torch.float16 else 64  # numbers from 1 to 1.5 that both types hold
    level = 1 + torch.randint(0, steps, (3000,), device="cuda", generator=case.g) / (2 * steps)
    level[::500] = 1 + torch.arange(6, device="cuda") / (2 * steps) + 0.5  # now and then a new largest
    case.keys = [(level[:, None, None] * 64).expand(3000, 1, 128).to(dtype).contiguous()]
    case.put(0, 0, case.keys[0], case.values[0])
    q = torch.full((new, 6, 128), 64.0, dtype=dtype, device="cuda")
    scale = 2.0 ** 25 / (64 * 64 * 128 * 2)
    out, lse = run_attention(P, case, q, scale=scale)
    first = 3000 - new
    for r in range(0, new, 37):
        seen = level[:first + r + 1]
        best = seen == seen.max()
        want = case.values[0][:first + r + 1, 0][best].double().mean(0)
        spread = case.values[0][:first + r + 1, 0][best].double().abs().mean(0)
        e = torch.finfo(dtype).eps / 2
        tol = e * want.abs() + spread * (e + 2.0 ** -20) * 1.01 + 2.0 ** -25
        assert torch.all((out[r].double() - want).abs() <= tol)
        top = scale * 64 * 64 * 128 * float(seen.max())
        assert torch.all((lse[r].double() - top).abs() <= top * 2.0 ** -15)


# ---- the tcgen05 kernels at the places where they can go wrong --------------------------------

def by_tiles(P, case, heads, window=0, slots=None):
    """Whether attention, or with `slots` the accumulated weight, takes the tcgen05 kernel."""
    L = P._bind()
    if slots is None:
        return bool(L.jfb_paged_attention_uses_tiles(case.rows, heads, window, case.cache.ref, case.batch.ref))
    return bool(L.jfb_paged_attention_mass_uses_tiles(case.rows, heads, case.cache.ref, case.batch.ref, C.c_uint64(slots)))


def check_masses_by_tiles(P, case, q, lse, scale, window, slots):
    before = torch.rand(len(case.kv), case.kvh, slots, device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    assert by_tiles(P, case, q.shape[1], window, slots)
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before, scale=scale, window=window, error_flag=case.error)
    torch.cuda.synchronize()
    # check_mass's bound, and what it leaves out: f32 has no normal number below 2^-126, so a term there may count as
    # zero, and a slot is off by up to 2^-126 more for each row and head
    for b, r, x, d, v in definition(case, q, scale, window):
        n, kv, G = case.new[b], case.kv[b], q.shape[1] // case.kvh
        seen = x > -math.inf
        l = torch.where(seen, lse[r].double().T[..., None], 0.0)
        p = torch.where(seen, torch.exp(x - l), 0.0)
        err = p * (2 * d + 2.0 ** -20 * (1 + x.abs().masked_fill(~seen, 0) + l.abs())) + 2.0 ** -126
        added = p.unflatten(0, (case.kvh, G)).sum((1, 2))
        old = before[b, :, :kv].double()
        old[:, max(0, kv - n):] = 0
        want = old + added
        tol = err.unflatten(0, (case.kvh, G)).sum((1, 2)) + added * U * (n * G + 8) + 2 * U * want
        assert torch.all((got[b, :, :kv].double() - want).abs() <= tol), b
    for b, k in enumerate(case.kv):
        assert torch.all(got[b, :, k:] == 9.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,kv,heads,kv_heads,hd,ps,window,pad,extra", [
    ([129, 7, 250], [2000, 900, 300], 5, 1, 64, 64, 0, 5, 20),
    ([512], [3000], 2, 2, 40, 32, 0, 0, 70),
    ([700, 1, 64], [2500, 40, 3000], 16, 2, 64, 16, 500, 3, 0),
    ([300], [1300], 16, 2, 24, 128, 0, 1, 0),
    ([333, 2], [5000, 700], 8, 1, 8, 8, 2000, 0, 0),
    ([401], [2600], 9, 3, 104, 16, 0, 2, 0),
    ([130, 0, 90], [3000, 17, 700], 256, 2, 64, 256, 0, 0, 0),    # 128 query heads share a kv head: one token a row tile
    ([260], [1500], 65, 1, 128, 64, 0, 0, 0)])                    # 65: the second half of a row tile is nearly empty
def test_tiles_by_shape(P, dtype, new, kv, heads, kv_heads, hd, ps, window, pad, extra):
    case = Case(P, new, kv, kv_heads, hd, ps, dtype, seed=hd + len(new), pad=pad, heads_first=len(kv) == 1, extra=extra)
    q = case.queries(heads)
    assert by_tiles(P, case, heads, window)
    workspace = P.attention_workspace()
    out, lse = run_attention(P, case, q, window, workspace=workspace)
    check_attention(case, q, out, lse, hd ** -0.5, window)
    again, lse2 = run_attention(P, case, q, window, workspace=workspace)
    assert torch.equal(out.nan_to_num(), again.nan_to_num()) and torch.equal(lse, lse2)
    check_masses_by_tiles(P, case, q, lse, hd ** -0.5, window, max(kv) + 5)
    assert int(case.error) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rising", [True, False])
def test_tiles_with_a_moving_maximum(P, dtype, hd, rising):
    """Every later key scores higher, so that each tile rescales the sums in tensor memory; or lower."""
    case = Case(P, [150], [2000], kv_heads=1, hd=hd, dtype=dtype, fill=False, extra=240)
    direction = rand(case.g, hd)
    direction /= direction.norm()
    ramp = torch.linspace(-30, 30, 2000, device="cuda")[:, None, None] * (1 if rising else -1)
    case.keys = [(direction * ramp).to(dtype).reshape(2000, 1, hd)]
    case.put(0, 0, case.keys[0], case.values[0])
    q = case.queries(6)
    q[:] = (direction * 40).to(dtype)
    assert by_tiles(P, case, 6)
    out, lse = run_attention(P, case, q, scale=0.1)
    check_attention(case, q, out, lse, 0.1, 0)
    check_masses_by_tiles(P, case, q, lse, 0.1, 0, 3000)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tiles_of_large_scores_and_constant_rows(P, dtype):
    case = Case(P, [200, 200], [600, 601], dtype=dtype, extra=70)
    q = case.queries(8, std=60.0)
    q[100] = 0
    assert by_tiles(P, case, 8)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)


@pytest.mark.parametrize("hd", [128, 72, 64, 40])
@pytest.mark.parametrize("odd", [0, 8])
def test_tiles_at_strides(P, hd, odd):
    """q a slice of a fused projection, out a slice of a wider buffer, on 32-byte sectors or 16 bytes off them."""
    heads = 12
    case = Case(P, [180, 180], [300, 555], hd=hd, pad=1, extra=60)
    fused = torch.full((case.rows, (heads + 4) * hd + odd), 3.0, dtype=case.dtype, device="cuda")
    q = fused[:, odd:odd + heads * hd]
    q.copy_(case.queries(heads).nan_to_num().reshape(case.rows, -1))
    wide = torch.full((case.rows, (2 + heads) * hd + odd), 7.0, dtype=case.dtype, device="cuda")
    out = wide[:, odd + hd:odd + (1 + heads) * hd].unflatten(1, (heads, hd))
    assert by_tiles(P, case, heads)
    out, lse = run_attention(P, case, q.unflatten(1, (heads, hd)), out=out)
    check_attention(case, q.unflatten(1, (heads, hd)), out, lse, hd ** -0.5, 0)
    assert torch.all(wide[:, :odd + hd] == 7.0) and torch.all(wide[:, odd + (1 + heads) * hd:] == 7.0)
    assert torch.all(fused[:, :odd] == 3.0) and torch.all(fused[:, odd + heads * hd:] == 3.0)


@pytest.mark.parametrize("hd", [128, 64])
def test_tiles_with_bad_pages(P, hd):
    """Pages outside the pool read as zeros and are flagged, by attention and by the accumulated weight."""
    case = Case(P, [140, 140], [400, 400], hd=hd, extra=300)
    case.table[0, 3] = -5
    case.table[1, 20] = case.k_pool.shape[0]
    case.table[1, 24] = 2 ** 31 - 1
    case.table[0, 25] = -1  # behind the keys: not read
    for b, page in ((0, 3), (1, 20), (1, 24)):
        case.keys[b][page * 16:page * 16 + 16] = 0
        case.values[b][page * 16:page * 16 + 16] = 0
    q = case.queries(8)
    assert by_tiles(P, case, 8)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, hd ** -0.5, 0)
    assert int(case.error) == P.ERROR_RANGE
    case.error.zero_()
    check_masses_by_tiles(P, case, q, lse, hd ** -0.5, 0, 2000)
    assert int(case.error) == P.ERROR_RANGE


@pytest.mark.parametrize("new,kv,extra", [([200], [60], 210), ([400, 3], [100, 0], 110)])
def test_tiles_of_rows_before_the_first_slot(P, new, kv, extra):
    case = Case(P, new, kv, extra=extra)
    q = case.queries(8)
    assert by_tiles(P, case, 8)
    out, lse = run_attention(P, case, q)
    check_attention(case, q, out, lse, 128 ** -0.5, 0)
    check_masses_by_tiles(P, case, q, lse, 128 ** -0.5, 0, 16 * case.width)
    assert int(case.error) == 0


@pytest.mark.parametrize("hd", [128, 64])
def test_tiles_of_masses_shorter_than_the_keys(P, hd):
    case = Case(P, [100, 100], [400, 150], hd=hd)
    heads, new = 32, 100
    q = case.queries(heads)
    out, lse = run_attention(P, case, q)
    before = torch.rand(2, 2, 170, device="cuda", generator=case.g)
    got = torch.full_like(before, 9.0)
    assert by_tiles(P, case, heads, slots=170)
    P.attention_mass(q, lse, case.cache, case.batch, got, mass_in=before, error_flag=case.error)
    wide = torch.full((2, 2, 400), 9.0, device="cuda")
    wide[:, :, :170] = before
    full = torch.full_like(wide, 9.0)
    P.attention_mass(q, lse, case.cache, case.batch, full, mass_in=wide)
    torch.cuda.synchronize()
    assert int(case.error) == P.ERROR_RANGE
    check_mass(case, q, lse, wide, full, hd ** -0.5, 0)
    # sums of the same positive terms, 16 a token and `before`, in an order that the cut may change
    assert torch.allclose(got, full[:, :, :170], rtol=2 * (16 * new + 8) * U, atol=0)
    assert torch.all(got[1, :, 150:] == 9.0)
