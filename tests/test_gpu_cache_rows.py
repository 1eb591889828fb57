"""ops.cache_write and ops.cache_read: rows of every type into caches of every
type against the definition in 64 bits, at the lengths, strides and positions
where they can go wrong, and their refusals (those run on the CPU too)."""

import math

import pytest
import torch

DEV = "cuda"
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOATS = [torch.float32, torch.bfloat16, torch.float16]
CODES = [torch.int8, torch.float8_e4m3fn]


def _ops():
    from multiscreen import ops
    return ops


def _name(t):
    return str(t).replace("torch.", "")


def nearest(t, ct):
    """The value of type ct nearest to float64 t, ties to the even one."""
    if ct == torch.int8:
        return t.round()
    grid = torch.exp2(torch.frexp(t).exponent.double() - 4).clamp(min=2.0 ** -9)
    return (t / grid).round() * grid


def quantised(x, ct):
    """(codes as float64 values, scale as float32) of rows x (..., D)."""
    top = x.double().abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top) & (top > 0)
    code = nearest(torch.where(ok, TOP[ct] * x.double() / torch.where(ok, top, 1.0), 0.0), ct)
    scale = torch.where(torch.isfinite(top), top.float() / torch.tensor(TOP[ct]), math.nan)
    return code, scale.squeeze(-1)


def empty_cache(B, cap, H, D, ct, device=DEV, fill=3):
    """Head-major caches and scales holding a known value everywhere."""
    k, v = (torch.full((B, H, cap, D), fill, dtype=torch.float32, device=device).to(ct).transpose(1, 2)
            for _ in range(2))
    if ct not in TOP:
        return k, v, None, None
    ks, vs = (torch.full((B, H, cap), 0.5, device=device).transpose(1, 2) for _ in range(2))
    return k, v, ks, vs


def rows_of(B, T, H, D, dt, seed=0):
    """k and v as two thirds of one stacked projection, rows of different lengths, with special rows."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, 3, H, D, generator=g) * torch.exp(torch.randn(B, T, 3, H, 1, generator=g))
    if T > 4:
        x[:, 1] = 0.0                                       # rows of zeros
        x[:, 2, :, :, 0] = math.inf
        x[:, 3, :, :, D - 1] = math.nan
        x[:, 4] = x[:, 4].abs().amax(-1, keepdim=True) * (torch.arange(D) % 5 - 2) / 2.0  # ties: half the largest
    if dt == torch.float32 and T > 6:
        x[:, 5] *= 1e-41                                    # subnormal rows
        x[:, 6] *= 1e36
    x = x.to(dt).to(DEV).view(B, T, 3 * H * D)
    return [x[:, :, i * H * D:(i + 1) * H * D].view(B, T, H, D) for i in (1, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("ct", CODES, ids=_name)
@pytest.mark.parametrize("dt", FLOATS, ids=_name)
@pytest.mark.parametrize("B,T,H,D", [(1, 1, 1, 16), (2, 7, 3, 32), (3, 65, 5, 64), (2, 130, 2, 128), (1, 2000, 8, 64)])
def test_codes_are_the_nearest(B, T, H, D, dt, ct):
    ops = _ops()
    k, v = rows_of(B, T, H, D, dt, seed=T)
    kc, vc, ks, vs = empty_cache(B, T + 9, H, D, ct)
    ops.cache_write(k, v, kc, vc, 4, ks, vs)
    back = ops.cache_read(kc, vc, ks, vs, 4, T, dt)
    for x, c, s, y in ((k, kc, ks, back[0]), (v, vc, vs, back[1])):
        code, scale = quantised(x.cpu(), ct)
        assert torch.equal(c[:, 4:4 + T].float().cpu().double(), code)
        # A/TOP in float32 is one rounding of the quotient
        assert torch.equal(s[:, 4:4 + T].cpu().nan_to_num(-1.0), scale.nan_to_num(-1.0))
        want = (code.float() * scale.unsqueeze(-1)).to(dt)  # exact codes, one fp32 product, one rounding
        assert torch.equal(y.cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))
        # the positions around stay as they were
        for part in (slice(0, 4), slice(4 + T, None)):
            assert (c[:, part].float() == 3).all() and (s[:, part] == 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", FLOATS, ids=_name)
def test_every_border_of_a_code(dt):
    """Values on and beside each border between two codes (rows of largest value TOP, so TOP x / A = x)."""
    ops = _ops()
    for ct in CODES:
        if ct == torch.int8:
            grid = torch.arange(-127.0, 128.0)
        else:
            grid = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
            grid = grid[torch.isfinite(grid)].sort().values
        mid = ((grid[1:] + grid[:-1]) / 2).to(dt)
        x = torch.cat((mid, torch.nextafter(mid.float(), torch.tensor(1e9)).to(dt),
                       torch.nextafter(mid.float(), torch.tensor(-1e9)).to(dt)))
        x = torch.cat((x, torch.zeros((-len(x)) % 63, dtype=dt))).view(-1, 63)
        x = torch.cat((x, torch.full((x.shape[0], 1), TOP[ct], dtype=dt)), 1)
        x = x.view(1, -1, 1, 64).to(DEV)
        kc, vc, ks, vs = empty_cache(1, x.shape[1], 1, 64, ct)
        ops.cache_write(x, -x, kc, vc, 0, ks, vs)
        for c, y in ((kc, x), (vc, -x)):
            assert torch.equal(c.float().cpu().double(), quantised(y.cpu(), ct)[0])
            assert ((ks == 1.0) & (vs == 1.0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ct", CODES + FLOATS, ids=_name)
def test_ragged_positions_rows_and_counts(ct):
    ops = _ops()
    dt = torch.bfloat16 if ct in TOP else ct
    B, Tx, H, D, cap, T = 4, 9, 3, 64, 40, 6
    k, v = rows_of(B, Tx, H, D, dt, seed=5)
    k, v = k.nan_to_num(1.0, 1.0, 1.0), v.nan_to_num(1.0, 1.0, 1.0)
    start = torch.tensor([0, 17, 38, -2], device=DEV)       # the third runs past the end, the last starts before 0
    rows = torch.tensor([[0, 2, 3, 5, 7, 8], [0, 1, -1, 9, 2, 3], [4, 5, 6, 7, 8, 0], [1, 2, 3, 4, 5, 6]], device=DEV)
    count = torch.tensor([6, 5, 4, 6], device=DEV)
    kc, vc, ks, vs = empty_cache(B, cap, H, D, ct)
    ops.cache_write(k, v, kc, vc, start, ks, vs, rows, count)
    one = empty_cache(B, Tx, H, D, ct)
    ops.cache_write(k, v, one[0], one[1], 0, one[2], one[3])  # every row's codes
    for x, c, s, src, ssrc in ((k, kc, ks, one[0], one[2]), (v, vc, vs, one[1], one[3])):
        want, wscale = torch.full((B, cap, H, D), 3.0), torch.full((B, cap, H), 0.5)
        for b in range(B):
            for t in range(int(count[b])):
                p, r = int(start[b]) + t, int(rows[b, t])
                if 0 <= p < cap and 0 <= r < Tx:
                    want[b, p] = src[b, r].float().cpu()
                    if s is not None:
                        wscale[b, p] = ssrc[b, r].cpu()
        assert torch.equal(c.float().cpu(), want)
        if s is not None:
            assert torch.equal(s.cpu(), wscale)
    # read back at the same ragged positions: zeros outside the cache
    got = ops.cache_read(kc, vc, ks, vs, start, T, dt)
    for b in range(B):
        for t in range(T):
            p = int(start[b]) + t
            for y, c, s in ((got[0], kc, ks), (got[1], vc, vs)):
                if not 0 <= p < cap:
                    assert (y[b, t] == 0).all()
                else:
                    ref = c[b, p].float() * (s[b, p].unsqueeze(-1) if s is not None else 1.0)
                    assert torch.equal(y[b, t], ref.to(dt))


@pytest.mark.gpu
def test_empty_calls_and_one_position():
    ops = _ops()
    kc, vc, ks, vs = empty_cache(2, 8, 2, 32, torch.int8)
    before = kc.clone()
    x = torch.randn(2, 0, 2, 32, device=DEV, dtype=torch.bfloat16)
    ops.cache_write(x, x, kc, vc, 8, ks, vs)
    assert ops.cache_read(kc, vc, ks, vs, 0, 0, torch.float32)[0].shape == (2, 0, 2, 32)
    far = torch.tensor([2 ** 62], device=DEV)  # one position for both sequences, far outside
    y = torch.randn(2, 3, 2, 32, device=DEV, dtype=torch.bfloat16)
    for s in (far, -far):
        ops.cache_write(y, y, kc, vc, s, ks, vs)
    ops.cache_write(y, y, kc, vc, 0, ks, vs, count=torch.tensor([0, -1], device=DEV))
    assert torch.equal(kc, before)


@pytest.mark.gpu
def test_a_cache_past_32_bit_offsets():
    """The last positions of a cache of over 2^32 bytes."""
    ops = _ops()
    B, cap, H, D = 1, 2 ** 22 - 1, 9, 128
    kc, ks = torch.zeros(B, H, cap, D, dtype=torch.int8, device=DEV), torch.zeros(B, H, cap, device=DEV)
    kc, ks = kc.transpose(1, 2), ks.transpose(1, 2)
    vc, vs = kc.clone(memory_format=torch.preserve_format), ks.clone(memory_format=torch.preserve_format)
    k, v = rows_of(B, 5, H, D, torch.bfloat16, seed=1)
    k, v = k.nan_to_num(1.0, 1.0, 1.0), v.nan_to_num(1.0, 1.0, 1.0)
    ops.cache_write(k, v, kc, vc, cap - 5, ks, vs)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        code, scale = quantised(x.cpu(), torch.int8)
        assert torch.equal(c[:, cap - 5:].cpu().double(), code) and torch.equal(s[:, cap - 5:].cpu(), scale)
        assert not c[:, :cap - 5].any() and not s[:, :cap - 5].any()


@pytest.mark.gpu
def test_write_and_read_replay_in_a_graph():
    ops = _ops()
    k, v = rows_of(2, 4, 2, 64, torch.float16, seed=3)
    kc, vc, ks, vs = empty_cache(2, 32, 2, 64, torch.int8)
    start = torch.zeros(2, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_write(k, v, kc, vc, start, ks, vs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_write(k, v, kc, vc, start, ks, vs)
        out = ops.cache_read(kc, vc, ks, vs, start, 4, torch.float16)
        start.add_(4)
    start.zero_()
    for step in range(6):
        k.normal_()
        v.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = empty_cache(2, 32, 2, 64, torch.int8)
        ops.cache_write(k, v, want[0], want[1], 4 * step, want[2], want[3])
        ref = ops.cache_read(*want, 4 * step, 4, torch.float16)
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1]), step
        assert torch.equal(kc[:, 4 * step:4 * step + 4], want[0][:, 4 * step:4 * step + 4])


@pytest.mark.gpu
def test_refusals():
    ops = _ops()
    x = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device=DEV)
    kc, vc, ks, vs = empty_cache(2, 8, 2, 64, torch.int8)
    cases = [
        (IndexError, (x, x, kc, vc, 6, ks, vs), {}),
        (IndexError, (x, x, kc, vc, -1, ks, vs), {}),
        (ValueError, (x, x, kc, vc, 0), {}),                                    # codes without scales
        (TypeError, (x, x, kc.float(), vc.float(), 0), {}),
        (ValueError, (x, x, x.new_zeros(2, 8, 2, 64), x.new_zeros(2, 8, 2, 64), 0, ks, vs), {}),
        (TypeError, (x, x.float(), kc, vc, 0, ks, vs), {}),
        (ValueError, (x, x, kc[:1], vc[:1], 0, ks[:1], vs[:1]), {}),
        (ValueError, (x, x, kc, vc, 0, ks.double(), vs.double()), {}),
        (ValueError, (x, x, kc, vc, torch.zeros(3, dtype=torch.int64, device=DEV), ks, vs), {}),
        (ValueError, (x, x, kc, vc, torch.zeros(2, dtype=torch.int32, device=DEV), ks, vs), {}),
        (ValueError, (x, x, kc, vc, 0, ks, vs), {"rows": torch.zeros(1, 3, dtype=torch.int64, device=DEV)}),
        (ValueError, (x, x, kc, vc, 0, ks, vs), {"count": torch.zeros(3, dtype=torch.int64, device=DEV)}),
        (RuntimeError, (x.cpu(), x.cpu(), kc, vc, 0, ks, vs), {}),
    ]
    for error, args, kw in cases:
        with pytest.raises(error):
            ops.cache_write(*args, **kw)
    odd = torch.zeros(2, 8, 2, 72, dtype=torch.int8, device=DEV)[..., :64]
    with pytest.raises(ValueError):
        ops.cache_write(x, x, odd, odd, 0, ks, vs)
    shared = kc[:1].expand(2, 8, 2, 64)
    with pytest.raises(_native_error()):  # two sequences would write one row
        ops.cache_write(x, x, shared, shared, 0, ks, vs)
    with pytest.raises(_native_error()):
        ops.cache_write(x, x, kc, vc, 0, ks[:1].expand(2, 8, 2), vs)
    # reading such a cache is fine
    assert ops.cache_read(shared, shared, ks, vs, 0, 8, torch.bfloat16)[0].shape == (2, 8, 2, 64)
    with pytest.raises(_native_error()):
        y = torch.zeros(2, 3, 2, 48, dtype=torch.bfloat16, device=DEV)
        c = torch.zeros(2, 8, 2, 48, dtype=torch.int8, device=DEV)
        ops.cache_write(y, y, c, c.clone(), 0, torch.zeros(2, 8, 2, device=DEV), torch.zeros(2, 8, 2, device=DEV))
    with pytest.raises(IndexError):
        ops.cache_read(kc, vc, ks, vs, 0, 9, torch.bfloat16)
    with pytest.raises(TypeError):
        ops.cache_read(kc, vc, ks, vs, 0, 2, torch.int8)


def _native_error():
    from multiscreen import _native
    return _native.MsaError


def test_c_entries_refuse_bad_arguments():
    """Argument checks run before any device work.  The pointers are no addresses, so this runs only where no
    kernel could start."""
    if torch.cuda.is_available():
        pytest.skip("a call that is not refused would start a kernel")
    from multiscreen import _native
    L = _native.lib()

    def pack(**kw):
        a = dict(k=16, ks=(512, 128, 64), B=2, T=3, Tx=3, H=2, D=64, dt=1, rows=0, count=0, start=0, n=0, s0=0,
                 c=16, cs=(1024, 64, 512), cap=8, ct=3, sc=16, ss=(16, 1, 8))
        a.update(kw)
        pair, cpair, spair = (a["k"], *a["ks"]), (a["c"], *a["cs"]), (a["sc"], *a["ss"])
        return _native.pack_cache_args(*pair, *pair, *cpair, *cpair, *spair, *spair, a["rows"], a["count"], a["start"], a["n"],
                                       a["s0"], a["B"], a["T"], a["Tx"], a["H"], a["D"], a["dt"], a["cap"], a["ct"])

    def write(**kw):
        return L.msa_cache_write(pack(**kw), None)

    for kw, msg in ((dict(D=48), "head_dim"), (dict(dt=3), "dtype"), (dict(ct=2), "cache_dtype"), (dict(ct=5), "cache_dtype"),
                    (dict(sc=0), "scales"), (dict(c=0), "null"), (dict(c=8), "aligned"), (dict(cs=(1024, 8, 512)), "multiples"),
                    (dict(k=0), "null"), (dict(ks=(512, 4, 64)), "strides"), (dict(T=4), "rows"), (dict(start=16, n=3), "start"),
                    (dict(ss=(16, -1, 8)), "strides"), (dict(cs=(0, 64, 512)), "share memory"), (dict(ss=(16, 0, 8)), "share memory"), (dict(B=70000, H=1), "B*H"), (dict(B=-1), "size"), (dict(T=2 ** 40), "size"), (dict(cs=(1024, 2 ** 26, 512)), "span")):
        assert write(**kw) == 1, kw
        assert msg in L.msa_last_error().decode(), (kw, L.msa_last_error())
    assert write(B=0) == 0 and write(T=0) == 0
    for kw, msg in ((dict(k=0), "k is null"), (dict(rows=16), "no rows"), (dict(count=16), "no rows"), (dict(T=4), "rows")):
        assert L.msa_cache_read(pack(**kw), None) == 1, kw
        assert msg in L.msa_last_error().decode(), (kw, L.msa_last_error())
    assert L.msa_cache_write(None, None) == 1 and b"args is null" in L.msa_last_error()
