"""More GPU checks of the window attention and 8-bit cache calls: scales that
are NaN, counts and workspaces that are refused, positions next to 2^31, runs
of many key tiles in one CTA."""
import pytest
import torch

from window_ref import D, SCALE_F16, attention64, check, fp8_cache, normal, values

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("splits", [1, 3, 20])
@pytest.mark.parametrize("row", [0, 100, 299])
def test_a_nan_value_scale_reaches_the_rows_that_see_it(grout, splits, row):
    """A cache row stands for code * scale: with a NaN scale every element of a
    value row is NaN, in attention as in the read-back.  Out of the window it
    is not seen."""
    hq, hkv, n, ps = 8, 2, 320, 64
    (kc, ks), (vc, vs) = (fp8_cache(s, n // ps, hkv, ps, D) for s in (10, 20))
    table = torch.arange(n // ps, dtype=torch.int32, device="cuda").view(1, -1)
    pos = _i32(299)
    q = normal(30, 1, hq, D).half()
    vs[row // ps, 1, row % ps] = NAN
    out = torch.empty_like(q)
    grout.attention_decode_paged_fp8(q, kc, vc, ks, vs, table, pos, out, n, num_splits=splits)
    ko, vo = (torch.empty(300, hkv, D, dtype=torch.float16, device="cuda") for _ in "kv")
    grout.kv_read_paged_fp8(kc, vc, ks, vs, table, ko, vo, _i32(0, 300))
    torch.cuda.synchronize()
    grout.check_device_error()
    assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all()
    assert torch.isnan(vo[row, 1]).all() and torch.isfinite(vo[row, 0]).all()
    if row == 100:
        grout.attention_decode_paged_fp8(q, kc, vc, ks, vs, table, pos, out, n, 199, 100, num_splits=splits)  # keys 101..299 and 0..99
        k, v = (values(c, s).transpose(1, 2).reshape(n, hkv, D)[:300] for c, s in ((kc, ks), (vc, vs)))
        v[row, 1] = 0.0
        check(out, *attention64(q, k, v, pos.long(), 199, 100, SCALE_F16))
