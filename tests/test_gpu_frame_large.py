"""Rows and items past the 2^32 threads that one launch may have: norms, rotations and appends of
tens of gigabytes, and attention calls that are refused whole."""
import pytest

pytestmark = pytest.mark.gpu

TILE = 1 << 16  # tokens that the inputs repeat


def repeats(big, tile):
    """Whether rows of `big` are `tile` again and again (the last time in part)."""
    import torch

    whole = len(big) // len(tile)
    for i in range(0, whole, 256):
        n = min(256, whole - i)
        if not torch.equal(big[i * len(tile):(i + n) * len(tile)].view(n, *tile.shape), tile.expand(n, *tile.shape)):
            return False
    rest = len(big) - whole * len(tile)
    return torch.equal(big[whole * len(tile):], tile[:rest])


def test_norm(gpu_ctx):
    """2^28 + 3 rows of 8 channels, 16 to a workgroup; a gate for each 2^26 rows."""
    import torch

    from jasnamacos_amd.frame_attention import GatedNorm

    print("case: norm of 2^28 rows", flush=True)
    tokens, run = (1 << 28) + 3, 1 << 26
    g = torch.Generator().manual_seed(1)
    tile = torch.randn(TILE, 8, generator=g).bfloat16().cuda()
    gate = torch.randn(5, 8, generator=g).bfloat16().cuda()
    x = tile.repeat(tokens // TILE + 1, 1)[:tokens]
    x_out = torch.empty_like(x)
    GatedNorm(gpu_ctx, 8, run).forward_dev(x, x, gate, None, None, x_out)
    norm, small = GatedNorm(gpu_ctx, 8, TILE), torch.empty_like(tile)
    for i in range(5):
        norm.forward_dev(tile, tile, gate[i:i + 1], None, None, small)
        torch.cuda.synchronize()
        assert repeats(x_out[i * run:(i + 1) * run], small), i


def test_rotary(gpu_ctx):
    """Five items a token (pairs and channels one by one: the rows are off 16 bytes), in place."""
    import torch

    from jasnamacos_amd.frame_attention import Rotary

    print("case: rotation of 2^32 items", flush=True)
    tokens = (1 << 32) // 5 + 70001
    g = torch.Generator().manual_seed(2)
    tile, positions = torch.randn(TILE, 1, 8, generator=g).half().cuda(), torch.randint(0, 99, (TILE, 3), generator=g).int().cuda()
    op = Rotary(gpu_ctx, 8, (1, 1, 1))
    freq, want = op.frequencies(), torch.empty_like(tile)
    op.run_dev(tile, positions, freq, want)
    room = torch.empty(tokens * 8 + 1, dtype=torch.float16, device="cuda")
    x = room[1:].view(tokens, 1, 8)
    places = torch.empty(tokens, 3, dtype=torch.int32, device="cuda")
    for i in range(0, tokens, 256 * TILE):
        n = min(256 * TILE, tokens - i)
        x[i:i + n] = tile.repeat(256, 1, 1)[:n]
        places[i:i + n] = positions.repeat(256, 1)[:n]
    op.run_dev(x, places, freq, x)
    torch.cuda.synchronize()
    assert repeats(x, want)
    del x, room, places


def test_append(gpu_ctx):
    """Eight items a token; one key and one value for all of them."""
    import torch

    from jasnamacos_amd.frame_attention import CacheAppend

    print("case: append of 2^32 items", flush=True)
    tokens, page = (1 << 29) + 77, 1 << 16
    width = -(-tokens // page)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(9, generator=g).half().cuda()[1:].view(1, 1, 8) for _ in range(2))
    pages = [torch.zeros(width, page, 1, 8, dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, width)
    cu, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, tokens], [tokens]))
    CacheAppend(gpu_ctx).run_dev(k.expand(tokens, 1, 8), v.expand(tokens, 1, 8), *pages, table, cu, lens)
    torch.cuda.synchronize()
    for got, one in zip(pages, (k, v)):
        rows = got.view(-1, 8)
        assert repeats(rows[:tokens], one.view(1, 8).repeat(TILE, 1)) and (rows[tokens:] == 0).all()


@pytest.mark.parametrize("dim", [64, 96])
def test_attention_too_large(dim, gpu_ctx):
    """65,535 sequences with a bound of 2^20 tokens each: an error, and nothing written."""
    import torch

    from jasnamacos_amd.deform_conv import DeformConvError
    from jasnamacos_amd.frame_attention import FrameAttention

    print("case: attention too large", dim, flush=True)
    op, tokens = FrameAttention(gpu_ctx, 1, 1, dim, back=8), 1 << 20
    q = torch.zeros(tokens, 1, dim, dtype=torch.bfloat16, device="cuda")
    outs = [torch.full_like(q, 7) for _ in range(4)]
    lse = torch.zeros(tokens, 1, device="cuda")
    cu = (torch.arange(65536, device="cuda") * 16).int()
    with pytest.raises(DeformConvError):
        op.forward_dev(q, q, q, outs[0], cu_q=cu, cu_kv=cu, max_q=tokens, max_kv=tokens)
    for bounds in ((tokens, 16), (16, tokens)):
        with pytest.raises(DeformConvError):
            op.backward_dev(q, q, q, q, lse, q, *outs[1:], cu_q=cu, cu_kv=cu, max_q=bounds[0], max_kv=bounds[1])
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in outs)
    op.forward_dev(q, q, q, outs[0], cu_q=cu, cu_kv=cu, max_q=16, max_kv=16)
    torch.cuda.synchronize()
    assert (outs[0][:65535 * 16] == 0).all() and (outs[0][65535 * 16:] == 7).all()
