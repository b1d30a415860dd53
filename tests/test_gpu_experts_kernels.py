"""Each kernel behind the experts' operators at the sizes and layouts where it can go wrong, on whole numbers whose results are exact."""
import numpy as np
import pytest

import experts_oracle as ref
from experts_oracle import upload
from test_gpu_experts import _sizes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,groups,n,k", [(2000, 3, 584, 544), (900, 5, 198, 288), (4000, 2, 4088, 800), (1500, 3, 1411, 320), (60, 6, 200, 512)])
def test_mxfp4_grouped_gemm_panels_of_all_groups(gpu, rows, groups, n, k):
    """Every group's matrix in the same panels, one behind the other, widths that no tile divides; the last panel ends with the last group."""
    Q, rng = gpu.MXFP4, np.random.default_rng(n)
    own, blocks = n + n % 2, -(-k // 32)
    offsets = _sizes_of(groups, rows, rng, 0.0)
    value = rng.choice(np.array([0, 2, 4, 8 + 2, 8 + 4], np.uint8), (rows + groups * own, 32 * blocks))
    value[:, k:] = 0
    scales = rng.integers(127, 130, (rows + groups * own, blocks)).astype(np.uint8)
    x = (np.where(value & 8, -1, 1) * ref.E2M1[value & 7] * np.exp2(np.repeat(scales.astype(np.float32), 32, 1) - 127))[:, :k].astype(np.float32)
    codes = (value[:, 0::2] | value[:, 1::2] << 4).astype(np.uint8)
    D = upload(gpu, np.full((rows, n), 99, np.float32))
    Q.grouped_gemm(upload(gpu, codes[:rows]), upload(gpu, ref.panels(scales[:rows], fill=255)), upload(gpu, codes[rows:]), upload(gpu, ref.panels(scales[rows:], fill=255)), D,
                   upload(gpu, offsets), rows=rows, groups=groups, n=n, k=k, d_type=np.float32, lds_w=groups * own, stride_w=own * codes.shape[1], stride_ws=8 * own)
    got, w = D.to_host().reshape(rows, n), x[rows:].reshape(groups, own, k)[:, :n]
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        assert np.array_equal(got[r], x[r] @ w[g].T), g
