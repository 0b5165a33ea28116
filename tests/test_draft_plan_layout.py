"""Draft plans: what ft_extend's kernels read of the table before the kernel ahead has ended stays away from what that kernel writes."""
import torch

import branch_cases
from ft_b200 import extend

LINE = 128 // 4      # ints of a cache line


def test_trees_words_share_no_cache_line_with_the_schedule():
    # the table may start at any 16 bytes: a line apart whatever the start
    rng = branch_cases.rng_of(0)
    for _ in range(300):
        cached, nodes, shared, window = branch_cases.random_step(rng)
        hq, hkv, d = rng.choice(((4, 4, 128), (8, 2, 64), (32, 8, 128), (16, 2, 256), (16, 1, 64)))
        seq = [c + n for c, n in zip(cached, nodes)]
        info, table, _, _ = extend.host_plan(seq, nodes, [r * 2000 for r in range(len(seq))], hq, hkv, d,
                                             rng.choice((torch.float16, torch.float32)), shared_prefixes=shared, window=window, draft=True)
        words = info.tile_tokens // 32
        first, end = info.sms_off, info.sms_off + 16 * info.num_sms
        for s in table[info.spans_off:info.spans_off + 8 * info.num_spans].reshape(-1, 8).tolist():
            lo, hi = info.extra_off + s[0], info.extra_off + s[0] + s[1] * words      # of the words that the tree decides
            assert hi + LINE - 1 <= first or end + LINE - 1 <= lo
