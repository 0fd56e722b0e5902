"""Rules of the kernels that no result shows when they are broken: what they break is an order that the hardware keeps
nearly always.  Checked on the kernels' source text."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "radeonflow_kernels_b200", "csrc")


def _text(path):
    """Source without comments."""
    with open(path) as f:
        s = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", s, flags=re.S)


def _closing(s, start, pair):
    depth = 0
    for i in range(start, len(s)):
        depth += (s[i] == pair[0]) - (s[i] == pair[1])
        if depth == 0:
            return i
    raise AssertionError("unbalanced " + pair)


def _kernels():
    """(file, kernel, parameter list, body) of every kernel."""
    out = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        s = _text(path)
        for m in re.finditer(r"__global__\s+void\s+(?:__\w+__\s*\((?:[^()]|\([^()]*\))*\)\s*)*(\w+)\s*\(", s):
            end = _closing(s, m.end() - 1, "()")
            body = s.index("{", end)
            out.append((os.path.basename(path), m.group(1), s[m.end():end], s[body:_closing(s, body, "{}") + 1]))
    return out


KERNELS = _kernels()
IDS = [f"{f}:{name}" for f, name, _, _ in KERNELS]


def test_every_kernel_is_found():
    n = sum(len(re.findall(r"__global__", _text(p))) for p in glob.glob(os.path.join(CSRC, "*.cu*")))
    assert len(KERNELS) == n and n > 10


@pytest.mark.parametrize("kernel", KERNELS, ids=IDS)
def test_commits_on_stage_barriers_are_waited_for(kernel):
    """A tcgen05.commit that frees a stage arrives on the stage's barrier by itself: the producer waits for the last ones, or
    they could arrive in shared memory that another CTA has taken over."""
    _, _, _, body = kernel
    if re.search(r"umma_commit\w*\(\s*empty_bar", body):
        assert re.search(r"finish_producer\((ok, it|loads_ok, loads), \w+, empty_bar\(0\)", body)


def test_a_scale_slot_is_given_back_by_its_readers():
    """The pair kernel's scale warps rewrite a slot behind a barrier on which the epilogue warps that read it have arrived
    with release semantics; the accumulator's hand-back (relaxed arrive, commit) orders no shared-memory read."""
    body = next(b for _, name, _, b in KERNELS if name == "fp8_gemm_pair_kernel")
    scales, epilogue = body[body.index("warp >= 2"):].split("setmaxnreg.inc", 1)
    assert scales.index("mbar_wait(scale_empty_bar(buf)") < scales.index("st_shared_v4(slot")
    assert "tmem_full_bar(buf), (q" not in scales
    assert epilogue.index("ld_shared_u32(my_scale") < epilogue.index("mbar_arrive(scale_empty_bar(buf))")


def test_dependent_launches_read_nothing_as_constant_data():
    """A kernel that may start before the one in front of it has finished waits for it and then reads what it wrote: with loads
    that the compiler cannot move in front of that wait.  (In files with such kernels, the helpers they call included.)"""
    waiting = [(f, name, params) for f, name, params, body in KERNELS if "griddep_wait()" in body]
    assert len(waiting) >= 8
    for f, name, params in waiting:
        assert not re.search(r"const[^,]*\*\s*__restrict__", params), (f, name)
    for f in {f for f, _, _ in waiting} | {"ptx.cuh", "fp8_tiles.cuh"}:
        assert not re.search(r"__ld(g|cg|ca|cs|lu)\(", _text(os.path.join(CSRC, f))), f


def test_dependent_launches_wait():
    """Files that launch kernels as programmatic dependents: each of their kernels waits, or is launched without."""
    plain = {"sort_count_kernel", "tile_list_kernel"}      # `launch(..., false, ...)`, <<< >>>
    for f, name, _, body in KERNELS:
        if "programmaticStreamSerializationAllowed" in _text(os.path.join(CSRC, f)) and name not in plain:
            assert body.count("griddep_wait()") == 1, (f, name)
    s = _text(os.path.join(CSRC, "moe_route.cu"))
    assert re.search(r"launch\(sort_count_kernel, [^;]*?, stream, false,", s) and "tile_list_kernel<<<" in s


def test_tables_have_arrived_before_anyone_is_told_of_them():
    """What the host writes for kernels of any stream goes through `upload`, which waits for the copy: cudaMemcpy from pageable memory
    and cudaMemset may return before, and a non-blocking stream is ordered behind neither."""
    for name in ("moe_few_api.cu", "moe_api.cu", "moe_ep_api.cu"):
        s = _text(os.path.join(CSRC, name))
        assert "rf::upload(" in s and not re.search(r"cudaMemcpy\w*\([^;]*HostToDevice", s), name
    s = _text(os.path.join(CSRC, "host_util.cu"))
    assert "cudaMemset(" not in s and "cudaStreamNonBlocking" in s and s.index("e = enqueue(s)") < s.index("cudaStreamSynchronize(s)")


def test_maps_in_device_memory_are_acquired():
    """Tensor maps that are no kernel parameters: the lane that issues the copies runs the tensor-map proxy's acquire fence on each
    before the first of them, and on the next one when the expert changes."""
    found = set()
    for f, name, params, body in KERNELS:
        if not re.search(r"p\.\w*maps\b", body):
            assert not re.search(r"CUtensorMap\s*\*", params), (f, name)
            continue
        pointers = re.findall(r"const CUtensorMap\* (m\w+) = (?!\()", body)
        for maps in pointers:
            loads = [m.start() for m in re.finditer(r"tma_load_\dd\w*\([^,]+, " + maps + r",", body)]
            if not loads or maps == "mx":           # (mx: the rows' maps, kernel parameters)
                continue
            found.add((name, maps))
            fence = body.index(f"tma_acquire_desc({maps})")
            assert re.search(r"if \((p\.maps != nullptr && )?m\w+ != acquired\) \{", body[:fence]) and fence < loads[0], (f, maps)
        # nor is one fetched before that
        assert not re.search(r"tma_prefetch_desc\((p\.|" + "|".join(pointers) + ")", body), f
    assert found == {("moe_few_kernel", "m0"), ("moe_few_kernel", "m1"), ("moe_gemm_kernel", "mw"), ("moe_gemm_kernel", "mw2")}


def test_grouped_scale_slots_are_given_back_after_they_were_read():
    """An arrival can overtake a shared-memory load that was issued before it: its address depends on what was loaded."""
    for kernel, arrival in (
            ("fp8_grouped_many_kernel", r"back = tmem_empty_bar\(buf\) \+ \(__float_as_uint\(s\) & \(\(uint32_t\)p\.groups >> 16\)\);"
                                        r".*if \(lane == 0\) mbar_arrive\(back\);"),
            ("fp8_grouped_few_kernel", r"mbar_arrive_after\(tmem_empty_bar\(buf\), seen, \(uint32_t\)p\.groups >> 16\)")):
        body = next(b for _, name, _, b in KERNELS if name == kernel)
        assert re.search(arrival, body, re.S) and "mbar_arrive(tmem_empty_bar" not in body, kernel
    # the mask is zero: at most 1024 groups
    assert re.search(r"kGroupedMaxGroups = 1024;", _text(os.path.join(CSRC, "fp8_grouped.cuh")))


def test_kernels_launched_through_the_helper_wait():
    """`launch_kernel(..., true, ...)` launches as a programmatic dependent: the same rule as above for the files that use it."""
    assert "programmaticStreamSerializationAllowed" in _text(os.path.join(CSRC, "launch.h"))
    through = [(f, name, body) for f, name, _, body in KERNELS if "launch_kernel(" in _text(os.path.join(CSRC, f))]
    assert {name for _, name, _ in through} >= {"quantize_rows_kernel", "quantize_blocks_kernel", "fp8_grouped_few_kernel",
                                                "fp8_grouped_many_kernel", "moe_few_kernel"}
    for f, name, body in through:
        assert body.count("griddep_wait()") == 1, (f, name)
        # nothing of another kernel's before it: what stands there are barriers, TMEM, indices and maps
        before = body[:body.index("griddep_wait()")]
        assert not re.search(r"ld_global|ld_word|atomic|tma_load|bulk_load|st_word", before), (f, name)
