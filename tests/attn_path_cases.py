"""Calls of attention over the paged cache, by the kernels they are meant to take.  test_attn_paths_host.py holds that they take them, the GPU tests their
results: a rule of the plan that moves one to other kernels fails there by name."""

F32, F16, Q4_0 = 0, 1, 2
KINDS = {F32: "f32", F16: "f16", Q4_0: "q4_0"}

# Units in shares, joined: heads that fill the registers and heads that do not, blocks of whole groups of 16 and of 4 positions and others; rows of a
# key-value head: up to eight, up to sixteen, two tiles of sixteen; all positions, a window with first tokens.  `kv` key-value heads.
SHARED = []
for type in (Q4_0, F16, F32):
    for dim in (32, 64, 96, 128, 192, 256):
        for block in (16, 20, 7):
            for group, new in ((4, 1), (9, 1), (8, 2), (20, 1)):
                if type != Q4_0 and (dim in (32, 192) or (block == 20 and group != 4)):
                    continue
                SHARED.append(dict(type=type, dim=dim, block=block, group=group, new=new, lens=[5200, 37, 3100] if (dim + block) % 3 else [4100], kv=1))
for c in SHARED:
    c.update(heads=c["group"] * c["kv"], heads_kv=c["kv"], seqs=len(c["lens"]), len=max(c["lens"]))

# Sequences that go in several parts, shares of each: short ones by the hundred, a few that are long.
PARTS = [dict(type=type, heads=8 * kv, heads_kv=kv, dim=dim, block=block, new=new, seqs=seqs, len=most)
         for type, dim, block, new, seqs, kv, most in ((Q4_0, 64, 16, 1, 300, 1, 6000), (Q4_0, 128, 20, 2, 300, 1, 5000), (Q4_0, 96, 7, 4, 270, 1, 5000),
                                                       (F16, 64, 16, 1, 300, 1, 6000), (F16, 128, 16, 4, 270, 1, 5000), (F32, 64, 7, 2, 520, 1, 3000))]

# Chosen blocks, as many units as compute units and more: whole, of several tiles of every wavefront.
LISTS_WHOLE = [dict(type=type, heads=group * kv, heads_kv=kv, dim=dim, block=block, seqs=2, new=rows, tokens=rows + 1, len=length, select=select)
               for type in (Q4_0, F16, F32)
               for dim, block, group, kv, rows, length, select in ((64, 16, 4, 4, 66, 1500, 40), (128, 20, 2, 3, 90, 1200, 33), (96, 7, 3, 2, 140, 1100, 100), (256, 16, 9, 2, 130, 900, 40),
                                                                   (128, 16, 20, 1, 131, 1000, 50))]
# Chosen blocks of few rows, in shares; and of many query heads a key-value head, which the many-row kernel takes.
LISTS_SHARED = [dict(type=type, heads=group, heads_kv=1, dim=dim, block=block, seqs=2, len=9000, select=select)
                for type in (Q4_0, F16, F32) for dim, block, group, select in ((64, 16, 4, 300), (128, 20, 9, 250), (96, 7, 8, 700), (256, 16, 20, 280))]
LISTS_MANY = [dict(type=type, heads=40, heads_kv=1, dim=dim, block=block, seqs=2, len=1200, select=select)
              for type in (Q4_0, F16, F32) for dim, block, select in ((64, 16, 40), (128, 7, 90))]
