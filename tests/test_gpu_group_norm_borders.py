"""group_norm_act where its forms meet: one workgroup an image and group holds up to 16384 values forward, 8192 (channels last) or 4096
(channels first) backward, and 1024 channels; test_train_ops_c_host.py says on which side of the border a size is.  The definition
and its bounds are those of test_gpu_group_norm.py."""
import pytest
import torch

from test_gpu_group_norm import ACTS, TYPES, check, make

pytestmark = pytest.mark.gpu

# channels of a group and positions: at 4096, 8192 and 16384 values, one position (or channel) less and more
BORDERS = [
    # one channel a group; odd numbers of positions are read one value at a time channels first
    (1, 4095), (1, 4096), (1, 4097), (1, 4100), (1, 8191), (1, 8192), (1, 8193), (1, 16383), (1, 16384), (1, 16385),
    # a few, and an odd few
    (4, 1023), (4, 1024), (4, 1025), (4, 2047), (4, 2048), (4, 2049), (4, 4095), (4, 4096), (4, 4097), (5, 819), (5, 820), (5, 1638), (5, 1639), (5, 3276), (5, 3277),
    (64, 64), (64, 65), (64, 128), (64, 129), (64, 256), (64, 257),
    # many channels and few positions: the most a workgroup's coefficients hold, and one more
    (1023, 1), (1024, 1), (1025, 1), (1023, 3), (1023, 4), (1024, 4), (1025, 4), (1023, 8), (1024, 8), (1023, 16), (1024, 16), (1025, 16), (1024, 17), (512, 32), (512, 33),
    # between the borders, where the launches have 512 and 1024 threads
    (7, 1500), (24, 515), (96, 150), (300, 54), (33, 333),
]


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
@pytest.mark.parametrize("dtype", TYPES, ids=("fp32", "bf16", "fp16"))
def test_on_both_sides_of_the_borders(genre, dev, dtype, last):
    for k, (cg, s) in enumerate(BORDERS):
        for n, groups in ((1, 2), (2, 1)):                                 # (one image writes its own dw and db, two add theirs up)
            act = ACTS[(k + n) % 4]
            print("border", cg, s, n, groups, dtype, last, act, flush=True)
            x, dy, w, b = make(dev, n, groups * cg, (s,), dtype, last, seed=k)
            check(genre, x, dy, w, b, groups, act)
