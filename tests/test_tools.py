"""The measurement scripts under tools/ are not run by the suite; this keeps them parseable."""
import glob
import os
import py_compile
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_python_tools_compile(tmp_path):
    files = sorted(glob.glob(os.path.join(ROOT, "tools", "*.py")))
    assert files
    for f in files:
        py_compile.compile(f, cfile=str(tmp_path / (os.path.basename(f) + "c")), doraise=True)


def test_shell_tools_parse():
    files = sorted(glob.glob(os.path.join(ROOT, "tools", "*.sh")))
    assert files
    for f in files:
        subprocess.run(["bash", "-n", f], check=True)


def test_counted_wait_scanner_flags_a_scalar_load_inside_the_region():
    """The attention and weight-gradient kernels wait for inline-asm LDS reads with counted lgkmcnt waits; the build
    fails if the compiler puts a scalar-memory instruction (which returns out of order on the same counter) between a
    transposed LDS read and the wait that drains the counter."""
    from vit_amd import build
    clean = """
_Z6kernelPv:
\tds_read_b64_tr_b16 v[0:1], v2 offset:0
\tds_read_b64_tr_b16 v[4:5], v2 offset:1024
\ts_waitcnt lgkmcnt(1)
\tv_mfma_f32_32x32x16_bf16 v[8:23], v[0:3], v[4:7], v[8:23]
\ts_waitcnt lgkmcnt(0)
\ts_load_dwordx2 s[0:1], s[4:5], 0x0
"""
    assert build.scan_counted_waits(clean) == []
    dirty = clean.replace("\ts_waitcnt lgkmcnt(1)\n", "\ts_load_dword s7, s[4:5], 0x10\n\ts_waitcnt lgkmcnt(1)\n")
    found = build.scan_counted_waits(dirty)
    assert len(found) == 1 and found[0][0] == "_Z6kernelPv" and "s_load_dword" in found[0][2]
    # a new kernel starts clean even if the previous one ended inside a region
    two = "_Z1aPv:\n\tds_read_b64_tr_b16 v[0:1], v2\n_Z1bPv:\n\ts_load_dword s0, s[4:5], 0x0\n\ts_waitcnt lgkmcnt(0)\n"
    assert build.scan_counted_waits(two) == []


def test_shipped_kernels_have_no_scalar_load_inside_counted_waits():
    from vit_amd import build
    assert build.check_counted_waits(verbose=False)


def test_in_flight_scanner_flags_uses_of_a_transposed_lds_read_before_its_wait():
    """The compiler takes the result of an inline-asm LDS read as there at once: a copy or a spill of it ahead of the wait
    moves whatever the register held."""
    from vit_amd import build
    clean = """
_Z6kernelPv:
\tds_read_b64_tr_b16 v[0:1], v2 offset:0
\tds_read_b64_tr_b16 v[4:5], v2 offset:1024
\tv_exp_f32_e32 v3, v3
\ts_waitcnt lgkmcnt(1)
\tv_mov_b64_e32 v[6:7], v[0:1]
\ts_waitcnt lgkmcnt(0)
\tv_mov_b32_e32 v9, v5
\ts_endpgm
.Lfunc_end0:
"""
    assert build.scan_in_flight(clean) == []
    copy = clean.replace("\tv_exp_f32_e32 v3, v3\n", "\tv_mov_b64_e32 v[6:7], v[0:1]\n")
    assert [ins for _, _, ins in build.scan_in_flight(copy)] == ["v_mov_b64_e32 v[6:7], v[0:1]"]
    spill = clean.replace("\tv_exp_f32_e32 v3, v3\n", "\tscratch_store_dwordx2 off, v[4:5], off offset:72\n")
    assert len(build.scan_in_flight(spill)) == 1
    early = clean.replace("lgkmcnt(1)", "lgkmcnt(2)")               # two reads on their way, one of them used
    assert len(build.scan_in_flight(early)) == 1
    younger = early.replace("\tv_exp_f32_e32 v3, v3\n", "\tds_read_b128 v[20:23], v2\n")
    assert build.scan_in_flight(younger) == []                       # two younger ones: lgkmcnt(2) covers the first
    # along a loop's back edge: the read at the end of the body is used at its start
    loop = ("_Z6kernelPv:\n.LBB0_1:\n\tv_add_u32_e32 v3, v0, v3\n\tds_read_b64_tr_b16 v[0:1], v2\n"
            "\ts_cbranch_vccnz .LBB0_1\n\ts_endpgm\n.Lfunc_end0:\n")
    assert len(build.scan_in_flight(loop)) == 1
    # an LDS-DMA that no wait has covered when its barrier comes
    dma = "_Z6kernelPv:\n\tglobal_load_lds_dwordx4 v[0:1], off\n\ts_waitcnt vmcnt({})\n\ts_barrier\n\ts_endpgm\n.Lfunc_end0:\n"
    assert build.scan_in_flight(dma.format(0)) == []
    assert len(build.scan_in_flight(dma.format(1))) == 1


def test_no_source_is_compiled_with_packed_f32_instructions():
    """Some forms of v_pk_add/mul/fma_f32 have given wrong results on this hardware."""
    from vit_amd import build
    pk = "_Z1aPv:\n\tv_pk_mul_f32 v[0:1], v[2:3], v[4:5]\n\tv_pk_add_bf16 v0, v1, v2\n\ts_endpgm\n.Lfunc_end0:\n"
    assert [ins.split()[0] for _, _, ins in build.scan_packed_f32(pk)] == ["v_pk_mul_f32"]
    assert build.check_counted_waits(verbose=False)
    flags = build.FLAGS
    at = flags.index("-packed-fp32-ops")
    assert flags[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]


def test_two_plane_representation_of_f32_round_trips_every_bit_pattern_class():
    """The residual stream between the folded blocks is held as plane H = upper half of bits(x) + 0x8000 (bf16 rounded
    half up) and plane L = lower half of bits(x); bits(x) = (H << 16) + sext16(L).  Host-side helpers (torch ops, the
    GPU epilogues write the same planes): exact on ties, carries, zeros, denormals, and plane H is the nearest bf16
    except that ties go up."""
    import torch
    from vit_amd import ops
    g = torch.Generator().manual_seed(3)
    bits = torch.randint(-2**31, 2**31 - 1, (200000,), generator=g, dtype=torch.int64).to(torch.int32)
    exp = (bits >> 23) & 0xFF
    bits = bits[exp != 0xFF]                                         # finite values
    special = torch.tensor([0, -2**31, 0x3F800000, 0x3F808000, 0x3F818000, 0x3F80FFFF, 0x3FFFFFFF, 0x00000001, 0x007FFFFF,
                            0x3F807FFF, 0x3F808001], dtype=torch.int64).to(torch.int32)
    x = torch.cat([bits, special]).view(torch.float32)
    h, lo = ops.f32_to_planes(x)
    assert h.dtype == torch.bfloat16 and lo.dtype == torch.bfloat16
    back = ops.planes_to_f32(h, lo)
    assert torch.equal(back.view(torch.int32), x.view(torch.int32))
    near = x.to(torch.bfloat16)                                      # round to nearest even
    tie = (x.view(torch.int32) & 0xFFFF) == 0x8000
    same = h.view(torch.int16) == near.view(torch.int16)
    big = ((x.view(torch.int32) >> 16) & 0x7FFF) >= 0x7F7F           # rounds to infinity either way: leave out
    assert bool((same | tie | big).all())
    up = (h.float() - x).abs() <= (near.float() - x).abs() * (1 + 1e-6) + 0.0
    assert bool((up | big | ~torch.isfinite(h.float())).all())       # never farther than the nearest bf16
