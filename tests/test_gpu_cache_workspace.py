"""One workspace for a whole decode: what vbs_cu_tree_workspace returns for
the longest context and the most tokens serves every shorter call."""
import pytest

pytestmark = pytest.mark.gpu

SHAPES = [(8, 4, 16, 128, 4672), (8, 8, 63, 128, 15040), (8, 4, 16, 128, 9000), (2, 4, 7, 64, 20000), (1, 8, 40, 96, 30000),
          (4, 4, 9, 256, 7000), (3, 5, 33, 80, 5000)]


def describe(vbs, nkh, group, tokens, hd, limit, max_ctx, ptr=4096, **kw):
    kv = vbs.KvDesc(k=ptr, v=ptr, n_layers=1, max_ctx=max_ctx, n_kv_heads=nkh, head_dim=hd, n_seqs=1, head_major=0)
    return kv, vbs.TreeDesc(n_q_heads=nkh * group, n_tokens=tokens, scale=1.0, ctx_limit=limit, n_ctx=ptr, **kw)


@pytest.mark.parametrize("nkh,group,tokens,hd,longest", SHAPES)
def test_the_query_grows_with_the_call(vbs, gpu, clean_errors, nkh, group, tokens, hd, longest):
    def need(limit, n, **kw):
        return vbs.tree_workspace(*describe(vbs, nkh, group, n, hd, limit, longest, **kw))

    for kw in (dict(), dict(window=700), dict(weights_out=4096)):
        last = 0
        for limit in range(64, longest + 1, 64):
            now = need(limit, tokens, **kw)
            assert now >= last, (limit, now, last)
            last = now
        last = 0
        for n in range(1, tokens + 1):
            now = need(longest, n, **kw)
            assert now >= last, (n, now, last)
            last = now
        assert need(longest, tokens, **kw) <= need(longest, tokens, **{**kw, "window": 0})


@pytest.mark.parametrize("nkh,group,tokens,hd,longest", SHAPES)
def test_the_longest_calls_workspace_serves_the_shorter(vbs, gpu, clean_errors, nkh, group, tokens, hd, longest):
    """Keys of zeros weigh every position the same, values count positions
    modulo head_dim: out[i][d] is the count of d over all that token i sees,
    to the halves' 2^-22 and a few roundings of 2^-24."""
    import torch
    k = torch.zeros((longest, nkh, hd), dtype=torch.float16, device="cuda")
    v = (torch.arange(longest, device="cuda")[:, None, None] % hd == torch.arange(hd, device="cuda")).expand(longest, nkh, hd).half().contiguous()
    q = torch.randn((tokens, nkh * group, hd), device="cuda")
    nbytes = vbs.tree_workspace(*describe(vbs, nkh, group, tokens, hd, longest, longest))
    work = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
    n_ctx = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = torch.arange(hd, device="cuda", dtype=torch.float64)
    for limit in list(range(longest, 63, -448)) + [64, tokens]:
        for n in sorted({1, 2, max(1, tokens // 2), tokens}):
            kv, tree = describe(vbs, nkh, group, n, hd, limit, longest)
            kv.k, kv.v, tree.n_ctx = k.data_ptr(), v.data_ptr(), n_ctx.data_ptr()
            n_ctx.fill_(limit - n)
            out = torch.full((n, nkh * group, hd), 7.0, device="cuda")
            torch.cuda.synchronize()
            vbs.attention_tree(kv, 0, tree, q.data_ptr(), out.data_ptr(), work.data_ptr(), nbytes)
            torch.cuda.synchronize()
            seen = torch.arange(limit - n + 1, limit + 1, device="cuda", dtype=torch.float64)[:, None]
            want = (((seen - d - 1) / hd).floor() + 1).clamp(min=0) / seen
            torch.testing.assert_close(out.double(), want[:, None].expand_as(out), rtol=2.0 ** -19, atol=0.0)
    gpu.synchronize_device(gpu.get_device(0))
    assert vbs.last_error() == "ok"
