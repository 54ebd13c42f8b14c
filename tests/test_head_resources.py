"""The compiler's report of the kernels of layer norm and of the unembedding's cross entropy (see ``test_kernel_resources``): what
they spill is known and does not grow, and their LDS fits."""
import glob
import os
import re

import pytest

from test_kernel_resources import CSRC, _kernels

HEAD = r"loss_logits_kernel|grad_logits_kernel|sum_kernel|out_kernel|dx_kernel|join_kernel|target_rows_kernel|pack_[wx]_kernel|loss_kernel|dbias_kernel|absmax_kernel|ln_"
# registers that do not fit, bytes a lane: all but those marked * lie outside of the loop over the rows or over k
KNOWN = {
    r"loss_logits_kernel.*TileILi4ELi2ELi2ELi4EEELb1ELb1EEE": (13, 48),  # fp32, 256 x 256
    r"ln_forward_kernelI\w+?Li4ELi1024ELi1024EEE": (95, 56),             # * 16-bit rows of more than 24576 elements
    r"ln_backward_kernelI\w+?Li2ELi(8|32|64)ELi1024EEE": (2, 12),        # 16-bit rows of up to 1024
    r"ln_backward_kernelIDF16_Li2ELi1024ELi1024EEE": (15, 64),           # * fp16 rows of more than 8192
    r"ln_backward_kernelIfLi4ELi(8|32|64)ELi1024EEE": (2, 12),           # fp32 rows of up to 1024
    r"ln_backward_kernelIfLi4ELi1024ELi1024EEE": (1, 8),                 # * fp32 rows of more than 12288
}


def _up_to_date():
    rules = glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(CSRC, "Makefile")]
    for name in ("layer_norm", "unembed"):
        report = os.path.join(CSRC, "build", name + ".remarks")
        if not os.path.exists(report):
            return False
        if os.path.getmtime(report) < max(os.path.getmtime(p) for p in [*rules, os.path.join(CSRC, name + ".hip")]) - 1:
            return False
    return True


@pytest.mark.skipif(not _up_to_date(), reason="no up-to-date build/*.remarks (make -C transcoder-sae-circuits_amd/csrc)")
def test_spills_of_the_heads_kernels_are_the_known_ones():
    head = {n: k for n, k in _kernels().items() if re.search(HEAD, n)}
    assert len(head) > 100, len(head)
    for pattern in KNOWN:
        assert any(re.search(pattern, n) for n in head), f"no such kernel: {pattern}"
    for n, k in head.items():
        registers, scratch = max((v for p, v in KNOWN.items() if re.search(p, n)), default=(0, 0))
        assert int(k["VGPRs Spill"]) <= registers and int(k["ScratchSize [bytes/lane]"]) <= scratch, (n, k)
        assert int(k["LDS Size [bytes/block]"]) <= 160 * 1024, (n, k)
