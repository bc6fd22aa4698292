"""Attention of many query rows over the same keys without a GPU: which way a call goes by its sizes, and what each refusal of the Python entry points says."""
import ctypes as C

import jittorinfer_amd as J
from tests.test_gqa_batch import _prefix


def test_prefixes_that_nobody_can_share_are_gqa_attn():
    """As many groups as sequences (what shared_prefixes gives a batch that shares nothing), one sequence alone: no row is there to be read once for two, whatever the
    table has room for.  One group fewer, and two sequences may share."""
    lib = J.library()
    size = lambda **kw: lib.gqa_prefix_attn_workspace_size(C.byref(_prefix(**kw)))
    for widths in (dict(), dict(dk=64, dv=64), dict(dk=256, dv=256)):
        for n_seq in (1, 2, 30):
            for stride in (4, 20000):
                call = dict(n_seq=n_seq, bt_stride=stride, **widths)
                alone = size(n_prefix=0, **call)
                for n_prefix in (n_seq, n_seq + 1, 3 * n_seq):
                    assert size(n_prefix=n_prefix, **call) == alone > 0
                if n_seq > 1 and stride == 20000:
                    assert size(n_prefix=n_seq - 1, **call) > alone
                assert size(n_prefix=n_seq, n_workgroups=16, **call) > size(n_prefix=0, n_workgroups=16, **call)
