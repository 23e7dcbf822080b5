"""Kernels of an overlapped chain (launch_pdl) start before the kernel ahead of them has written its output. Checked in the
sources, without a GPU: what another kernel wrote is read by accesses that stay behind pdl_wait(). Loads that promise data nothing
writes during the launch (__ldg, ld.global.nc, const __restrict__ parameters) or that carry no order (__ldcg) are for
weights, tables and norms."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "naiwa-rs_b200", "csrc")


def text_of(path):
    text = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def chain_files():
    names = [p for p in glob.glob(os.path.join(CSRC, "*.cu")) if "pdl_wait()" in text_of(p)]
    headers = [os.path.join(CSRC, h) for h in ("expert_frag.cuh", "attention_internal.cuh", "layer_internal.cuh")]
    return sorted(names) + headers


def kernels(text):
    """(name, parameters, body) of every __global__ function that waits for the kernel ahead of it."""
    found = []
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        params, start = text[m.end():i - 1], text.index("{", i)
        depth, j = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[j], 0)
            j += 1
        if "pdl_wait()" in text[start:j]:
            found.append((m.group(1), params, text[start:j]))
    return found


def test_every_chain_file_is_seen():
    names = {os.path.basename(p) for p in chain_files()}
    assert {"plan.cu", "router.cu", "expert_decode.cu", "expert_stream.cu", "expert_gemm_tc.cu", "attention.cu",
            "attention_decode.cu", "attention_prefill.cu", "expert_frag.cuh"} <= names
    assert sum(len(kernels(text_of(p))) for p in chain_files()) >= 14


# What never changes while a kernel runs: expert weights and their scales, router weights, rotary table, norm weights.
CONSTANT = re.compile(r"\s*(qb\b|sb\b|p\.wq\b|p\.wscale\b|wa\b|wb\b|wr\b|row \+ i\)|"
                      r"reinterpret_cast<const \w+\*>\((nw|p\.rope_table)\b)")


@pytest.mark.parametrize("path", chain_files(), ids=os.path.basename)
def test_unordered_loads_read_constants_only(path):
    text = text_of(path)
    for m in re.finditer(r"\b(__ldg|__ldcg|__ldca|__ldcs|ldg_nc|ldg_stream)\(", text):
        line = text[m.start():text.index("\n", m.start())]
        assert m.group(1) != "__ldcg" and CONSTANT.match(text, m.end()), line
    nc = [line for line in text.splitlines() if "ld.global.nc" in line]
    assert len(nc) == (1 if path.endswith("expert_frag.cuh") else 0), nc  # the 8-byte scales of one weight format


@pytest.mark.parametrize("path", chain_files(), ids=os.path.basename)
def test_parameters_of_chain_kernels_are_not_promised_constant(path):
    for name, params, _ in kernels(text_of(path)):
        assert "__restrict__" not in params, name


@pytest.mark.parametrize("path", chain_files(), ids=os.path.basename)
def test_no_cta_leaves_before_it_has_waited(path):
    """A kernel none of whose CTAs waits would complete ahead of the kernel before it."""
    for name, _, body in kernels(text_of(path)):
        before = body[:body.rindex("pdl_wait()")]
        for m in re.finditer(r"\breturn\b[^;]*;", before):
            assert re.search(r"pdl_leave\(\);\s*$", before[:m.start()]), (name, before[m.start() - 80:m.end()])


def test_the_decode_kernel_reads_its_record_once():
    """Threads that saw different records would use shared memory that the others never wrote."""
    body = dict((n, b) for n, _, b in kernels(text_of(os.path.join(CSRC, "expert_decode.cu"))))["expert_gemv_kernel"]
    head = body[:body.index("s_rec = r;")]
    assert "if (threadIdx.x == 0) {" in head and "act_rec" not in body[body.index("s_rec = r;"):]
    assert not re.search(r"p\.(n_active|active|offsets|slot_of)\b", body[body.index("s_rec = r;"):])


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu*"))), ids=os.path.basename)
def test_loads_in_assembly_are_volatile(path):
    """A load in a plain asm is a pure function to the compiler, which may evaluate it ahead of the test that guards it."""
    for m in re.finditer(r"\basm\s*(volatile\s*)?\(\s*\"([^;]*);", text_of(path)):
        assert m.group(1) or not re.search(r"\b(ld|ldu|ldmatrix|cp|tcgen05|atom|red|st)\b", m.group(2)), m.group(0)


def test_prefill_reads_its_error_word_once():
    """Threads of a CTA that saw different words would part before its barriers and its collective allocation."""
    body = dict((n, b) for n, _, b in kernels(text_of(os.path.join(CSRC, "attention_prefill.cu"))))["prefill_kernel"]
    reads = [m.start() for m in re.finditer(r"p\.err\)\s*==", body)]
    assert len(reads) == 1 and re.search(r"if \(tid == 0\) s_abort = [^;]*$", body[:reads[0]].rstrip("*"))
    assert body.index("__syncthreads();", reads[0]) < body.index("tcgen05.alloc")
    stop = body[reads[0]:body.index("tcgen05.alloc")]
    assert "leave();" in stop, "a CTA that leaves early counts itself"


def test_a_commit_follows_an_mma():
    """No commit in a CTA that has issued no MMA, and none whose arrival nothing waits for."""
    body = dict((n, b) for n, _, b in kernels(text_of(os.path.join(CSRC, "attention_prefill.cu"))))["prefill_kernel"]
    at = body.index("commit(&bars.drained)")
    assert "if (committed & 0x55)" in body[at - 120:at]


def test_the_grouped_gemm_reads_its_error_word_once():
    """As above: before the CTA's first barrier, by one thread."""
    body = dict((n, b) for n, _, b in kernels(text_of(os.path.join(CSRC, "expert_gemm_tc.cu"))))["expert_gemm_kernel"]
    assert not re.search(r"MOE_ERR_TIMEOUT\)\s*return", body)
    read = body.index("p.err) ==")
    assert "if (threadIdx.x == 0) s_abort = " in body[read - 90:read]
    assert "__syncthreads();" in body[read:body.index("if (s_abort) return;")] and body.count("s_abort = 0") == 0


def test_no_device_wide_limit_is_changed():
    """A limit of the context is its other users' too (a stack reserve of 16 KB per thread held 5 GB of the device)."""
    for path in glob.glob(os.path.join(CSRC, "*.c*")):
        assert "DeviceSetLimit" not in text_of(path) and "CtxSetLimit" not in text_of(path), path


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu*"))), ids=os.path.basename)
def test_loads_of_what_others_write_are_ordered(path):
    """__ldcg carries no order against a wait, nor against the test that guards it: what a peer or another CTA wrote is read by
    ld_l2."""
    assert "__ldcg(" not in text_of(path)
