"""csrc/qd_tree.h's tree_attn_plan, restated: which blocks, splits and rounds a call takes."""


def attention_plan(nodes, heads, kv_heads, prefix, cus):
    """(block_rows, key_waves, blocks, splits, rounds, most splits)"""
    rows = nodes * (heads // kv_heads)
    wide = (rows + 127) // 128 * 2 == (rows + 63) // 64
    block_rows = 16 if rows <= 16 else 32 if rows <= 32 else 128 if wide else 64
    key_waves = 8 if rows <= 32 else 2 if wide else 4
    blocks = -(-rows // block_rows)
    most = max(1, cus // (blocks * kv_heads))
    groups = -(-(-(-prefix // 32) + -(-nodes // 32)) // key_waves)
    rounds = -(-groups // most)
    splits = -(-groups // rounds)
    if groups <= (3 if key_waves == 8 else 2):
        splits, rounds = 1, groups
    return block_rows, key_waves, blocks, splits, rounds, most
