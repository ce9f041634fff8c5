"""The groups of the serving ops that the tests prebuild: every type, format,
head layout, block size and schedule of each."""
from hfusion_mi355x import groups as g

_ANY = 7919

# rows, cols, element type, type of the weight, codes, residual
NORM = [
    (3, 1, "f32", "f32", "i8", True), (5, 7, "bf16", "f32", "e4m3", False), (9, 64, "f16", "f16", "i8", True), (6, 33, "f32", "f32", "e5m2", True),
    (33, 512, "bf16", "bf16", "i8", True), (130, 1000, "bf16", "bf16", "e4m3", True), (40, 1024, "f16", "f32", "e5m2", False),
    (7, 1032, "f32", "f32", "i8", False), (700, 2001, "bf16", "f32", "i8", True), (5, 4096, "bf16", "bf16", "e4m3", True),
    (3, 5003, "f32", "f32", "i8", True), (2, 8200, "bf16", "f32", "e4m3", True), (2, 16384, "f16", "f32", "i8", True),
    (600, 320, "f32", "f32", "e4m3", True), (1, 16383, "f32", "f32", "e5m2", True), (2100, 96, "bf16", "bf16", "i8", False),
]
# heads, kv heads, dim, block, slots, room, blocks, element type, format
APPEND = {
    "group4": (8, 2, 64, 16, 5, 160, 40, "bf16", "e4m3"), "alone": (4, 4, 32, 16, 3, 64, 13, "f32", "e5m2"),
    "group3": (6, 2, 96, 32, 4, 320, 30, "f16", "e4m3"), "wide": (4, 1, 256, 128, 3, 512, 11, "bf16", "e5m2"),
    "usual": (32, 8, 128, 64, 6, 640, 40, "bf16", "e4m3"), "many": (2, 1, 32, 16, 700, 64, 2900, "bf16", "e4m3"),
}
# rotated channels, neighbouring pairs
TURN = {"group4": (64, 0), "alone": (32, 1), "group3": (48, 0), "wide": (128, 1), "usual": (128, 0), "many": (32, 0)}
# the same for the attention, and its window
ATTEND = {
    "group4": (8, 2, 64, 16, 5, 160, 40, "bf16", "e4m3", 0), "alone": (4, 4, 32, 16, 5, 160, 47, "f16", "e5m2", 0),
    "group3": (6, 2, 96, 32, 5, 320, 40, "f16", "e4m3", 0), "group32": (32, 1, 128, 64, 5, 640, 40, "bf16", "e4m3", 0),
    "group20": (20, 1, 64, 32, 5, 320, 40, "bf16", "e5m2", 0), "wide": (4, 1, 256, 128, 5, 512, 20, "bf16", "e5m2", 0),
    "window": (8, 2, 64, 32, 5, 640, 90, "bf16", "e4m3", 50), "window_f16": (4, 2, 128, 16, 5, 320, 90, "f16", "e4m3", 7),
    "usual": (32, 8, 128, 64, 6, 4096, 90, "bf16", "e4m3", 0), "far": (8, 2, 128, 16, 3, 8192, 600, "bf16", "e4m3", 0),
    "far_f16": (6, 2, 96, 32, 3, 4096, 300, "f16", "e4m3", 0), "far_group20": (20, 1, 64, 64, 3, 4096, 150, "bf16", "e5m2", 0),
    "far_window": (8, 2, 64, 16, 3, 4096, 600, "bf16", "e4m3", 1500), "far_wide": (4, 1, 256, 128, 3, 4096, 80, "f16", "e5m2", 0),
    "far_alone": (3, 3, 32, 32, 3, 4096, 300, "bf16", "e4m3", 0), "many": (2, 1, 32, 16, 150, 4096, 2900, "bf16", "e4m3", 0),
    "far_longer": (8, 2, 64, 16, 3, 4096, 600, "f16", "e4m3", 2500), "wide_f16": (4, 2, 192, 32, 3, 2048, 300, "f16", "e4m3", 0),
}
# rows of the groups that are compiled for one row count
STATIC = {"append": ("usual", 70), "attend": ("usual", 70)}
# a decoder layer's attention: columns of the residual stream, its cache
# the un-fused layer as a program
PROGRAM = dict(rows=20, cols=512, heads=8, kv_heads=2, dim=64, slots=4, room=4096, blocks=300, block=32)
# a cache whose last blocks lie past byte 2^31, and a small one
BIG = dict(rows=130, heads=8, kv_heads=8, dim=128, slots=2, room=192, blocks=33000, block=64, few=8)
LAYER = dict(cols=512, heads=8, kv_heads=2, dim=64, slots=4, room=256, blocks=24, block=32)


def norm_name(c):
    r, n, el, p, out, res = c
    return f"rmsnorm_{out}_{el}_{p}_{r}x{n}_{'r' if res else 'x'}"


def norm(rows, cols, elem, params, out, residual, **kw):
    return g.rms_norm(rows, cols, elem=elem, params=params, out=out, residual=residual, **kw)


def _sizes(c):
    hq, hk, d, block, slots, room, blocks, el, fmt = c[:9]
    return dict(heads=hq, kv_heads=hk, dim=d, block=block, slots=slots, room=room, blocks=blocks, elem=el, fmt=fmt)


def append(name, rows):
    rot, pairs = TURN[name]
    return g.append_kv(rows, rot=rot, pairs=bool(pairs), **_sizes(APPEND[name]))


def attend(name, rows):
    return g.paged_attention(rows, window=ATTEND[name][9], **_sizes(ATTEND[name]))


def norm_rank3():
    """[2, 3, 64]: the leading dims are the rows."""
    return g.rms_norm(6, 64).replace("<6x64x", "<2x3x64x").replace("<6xf32>", "<2x3xf32>")


def entries():
    rt = lambda ir: g.with_dynamic_rows(ir, _ANY)  # noqa: E731
    e = {norm_name(c): norm(*c) for c in NORM}
    e["rmsnorm_rank3"] = norm_rank3()
    e["rmsnorm_eps0"] = g.rms_norm(6, 100, eps=0.0)
    e["rmsnorm_i8_rt"] = rt(g.rms_norm(_ANY, 1000))
    e["rmsnorm_e4m3_rt"] = rt(g.rms_norm(_ANY, 4096, out="e4m3", params="f32"))
    e.update({f"appendkv_{n}_rt": rt(append(n, _ANY)) for n in APPEND})
    e.update({f"pagedattn_{n}_rt": rt(attend(n, _ANY)) for n in ATTEND})
    e["appendkv_static"] = append(*STATIC["append"])
    e["pagedattn_static"] = attend(*STATIC["attend"])
    layer = {k: v for k, v in LAYER.items() if k != "cols"}
    e["layer_norm_i8_rt"] = rt(g.rms_norm(_ANY, LAYER["cols"]))
    e["layer_qkv_rt"] = rt(g.w8a8_dequant(_ANY, (LAYER["heads"] + 2 * LAYER["kv_heads"]) * LAYER["dim"], LAYER["cols"]))
    e["layer_append_rt"] = rt(g.append_kv(_ANY, **layer))
    e["layer_attend_rt"] = rt(g.paged_attention(_ANY, **layer))
    size = {k: v for k, v in PROGRAM.items() if k not in ("rows", "cols")}
    rows, cols = PROGRAM["rows"], PROGRAM["cols"]
    e["prog_decoder_attention"] = g.decoder_attention(**PROGRAM)
    e["part_norm"] = g.rms_norm(rows, cols, out="e4m3")
    e["part_product"] = g.matmul_mx(rows, (size["heads"] + 2 * size["kv_heads"]) * size["dim"], cols, out="bf16")
    e["part_append"], e["part_attend"] = g.append_kv(rows, **size), g.paged_attention(rows, **size)
    big = {k: v for k, v in BIG.items() if k not in ("rows", "few")}
    for name, blocks in (("big", BIG["blocks"]), ("small", BIG["few"])):
        e[f"appendkv_{name}"] = g.append_kv(BIG["rows"], **{**big, "blocks": blocks})
        e[f"pagedattn_{name}"] = g.paged_attention(BIG["rows"], **{**big, "blocks": blocks})
    for name, scale in (("negative", -0.2), ("zero", 0.0), ("large", 3.0)):
        e[f"pagedattn_{name}_rt"] = rt(g.paged_attention(_ANY, scale=scale, **_sizes(ATTEND["group4"])))
    from norm_mx_catalog import untied
    e["pagedattn_untied"], e["rmsnorm_untied"] = untied(attend("usual", 70)), untied(g.rms_norm(33, 512))
    return e
