"""Score attention over the longest ranges of keys that are taken, 2^30, against float64 over those that are seen."""
from __future__ import annotations

import pytest
import torch

import flash_attention_amd as fa

pytestmark = pytest.mark.gpu


def test_documents_in_the_longest_range_of_keys():
    """4200 queries of one document, whose tokens lie at both ends of 2^30 (36 GiB of keys, values and ids)."""
    n, sq, d, ends = 1 << 30, 4200, 8, (50, 90)
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("60 GiB of device memory")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.zeros(n, d, dtype=torch.float16, device="cuda") for _ in range(2))
    ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    for part in (slice(0, ends[0]), slice(n - ends[1], n)):
        k[part] = torch.randn(k[part].shape, generator=g, device="cuda").half()
        v[part] = torch.randn(v[part].shape, generator=g, device="cuda").half()
        ids[part] = 5
    ids[1000:1100] = 0   # another document
    q = torch.randn(sq, d, generator=g, device="cuda").half()
    qids = torch.full((sq,), 5, dtype=torch.int32, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full((sq,), 7.0, device="cuda")
    c = fa.score_config(fa.DTYPE_F16, 1, 1, 1, sq, n, d, q_doc_ptr=qids.data_ptr(), k_doc_ptr=ids.data_ptr())
    fa.score_attention_device(c, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    seen = torch.cat((torch.arange(ends[0]), torch.arange(n - ends[1], n))).cuda()
    z = q.double() @ k[seen].double().t().contiguous() / d ** 0.5
    want = torch.softmax(z, 1) @ v[seen].double()
    # weights and result are rounded once each (2^-11), f32 errors are far below a quarter of that
    assert (out - want).abs().max() <= 2.25 * 2.0 ** -11 * v[seen].double().abs().max()
    assert (lse - torch.logsumexp(z, 1)).abs().max() <= 1e-4
    del k, v, ids
    torch.cuda.empty_cache()
