"""Further groups of the attention that the tests prebuild: windows over blocks of
64 and 128 tokens, in both types, and f16 heads in groups of more than 16.  Fields as serving_catalog.ATTEND's."""
import serving_catalog as sc
from hfusion_mi355x import groups as g

ATTEND = {
    "window_f16_64": (1, 1, 64, 64, 5, 1024, 90, "f16", "e4m3", 100), "window_f16_128": (8, 2, 128, 128, 5, 1024, 45, "f16", "e5m2", 300),
    "window_64": (8, 2, 64, 64, 5, 1024, 90, "bf16", "e4m3", 100), "window_128": (6, 2, 96, 128, 5, 1024, 45, "bf16", "e5m2", 30),
    "far_window_f16_64": (8, 2, 64, 64, 3, 4096, 200, "f16", "e4m3", 2500), "far_window_f16_128": (3, 3, 256, 128, 3, 4096, 100, "f16", "e4m3", 1100),
    "group20_f16": (20, 1, 64, 16, 5, 320, 90, "f16", "e5m2", 0), "far_group20_f16": (40, 2, 96, 32, 3, 4096, 300, "f16", "e4m3", 0),
}


def entries():
    return {f"pagedattn_{n}_rt": g.with_dynamic_rows(g.paged_attention(7919, window=c[9], **sc._sizes(c)), 7919) for n, c in ATTEND.items()}
