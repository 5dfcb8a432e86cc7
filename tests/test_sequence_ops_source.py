"""Rules of the device code that no run can be relied on to show (a violation
is a race that may never fire on one GPU): read from the sources, no GPU."""

import glob
import os
import re

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = sorted(glob.glob(os.path.join(REPO, "macmetalpy_b200", "csrc", "*.cu"))
                 + glob.glob(os.path.join(REPO, "macmetalpy_b200", "csrc", "*.cuh")))


def kernels(path):
    """{name: (parameters, body)} of a file's __global__ functions, comments taken out."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)

    def until(at, opening, closing):
        depth = 0
        while True:
            depth += (text[at] == opening) - (text[at] == closing)
            at += 1
            if depth == 0:
                return at

    found = {}
    for m in re.finditer(r"__global__", text):
        at = m.end()
        while True:  # attributes in parentheses, then the name and its parameters
            paren = text.index("(", at)
            end = until(paren, "(", ")")
            name = re.search(r"(\w+)\s*$", text[at:paren]).group(1)
            if not name.startswith("__"):
                break
            at = end
        brace = re.match(r"\s*\{", text[end:])
        if brace:
            found[name] = (text[paren + 1:end - 1], text[end + brace.end() - 1:until(end + brace.end() - 1, "{", "}")])
    return found


ALL = {(os.path.basename(p), name): parts for p in SOURCES for name, parts in kernels(p).items()}


def test_the_kernels_are_found():
    for name in ("emb_sort_kernel", "emb_sum_kernel", "rec_kernel", "norm_sum_kernel", "scan_tiles_kernel"):
        assert [k for k in ALL if k[1] == name], name


SENDS = r"map_shared_rank|rec_send\s*\(|mapa\."
WAITS = r"\bsync\s*\(\s*\)\s*;|barrier_wait\s*\(|barrier\.cluster\.wait"


def cluster_sync(body):
    """Position of the first wait of the whole cluster (its own barrier, not __syncthreads or __syncwarp)."""
    for m in re.finditer(WAITS, body):
        if m.group(0).startswith("sync") and not re.search(r"\bcl(uster)?\.$", body[:m.start()]):
            continue
        return m.start()
    return len(body)


@pytest.mark.parametrize("kernel", [k for k, v in ALL.items() if re.search(SENDS, v[1])], ids="/".join)
def test_shared_memory_of_other_blocks_after_a_cluster_barrier(kernel):
    """A block's shared memory may be reached by others only once it is known
    to run: a barrier of the whole cluster comes before the first access."""
    body = ALL[kernel][1]
    assert cluster_sync(body) < re.search(SENDS, body).start()


CHAINED = [p for p in SOURCES if "chain_wait();" in open(p).read()]


@pytest.mark.parametrize("path", CHAINED, ids=os.path.basename)
def test_chained_kernels_promise_nothing_of_their_inputs(path):
    """A kernel that is set up while its predecessor still writes must not tell
    the compiler that its inputs stay as they are: loads marked so (const
    __restrict__, __ldg, ld.global.nc) need not stay behind the wait."""
    text = re.sub(r"//[^\n]*", "", open(path).read())
    assert not re.findall(r"const\s+[\w:<>, ]+\*\s*__restrict__[^,)]*", text)
    assert "__ldg" not in text and "ld.global.nc" not in text


def test_files_of_chained_kernels_are_found():
    assert {"mmp_embedding.cu", "mmp_norm.cu", "mmp_recurrence.cu"} <= {os.path.basename(p) for p in CHAINED}


@pytest.mark.parametrize("path", [p for p in SOURCES if "cudaFuncSetAttribute" in open(p).read()], ids=os.path.basename)
def test_limits_of_shared_memory_are_set_once(path):
    """A kernel's limit of dynamic shared memory is set once per device: set
    anew by every call, another thread's call could lower it between this
    one's setting and its launch."""
    lines = open(path).read().splitlines()
    for i, line in enumerate(lines):
        if "cudaFuncSetAttribute(" in line:
            assert any(re.search(r"if \(!\w+\[dev\]", before) for before in lines[max(0, i - 5):i]), (i + 1, line)


def test_the_embedding_gradients_sort_keeps_nothing_between_calls():
    """mmp_scan keeps look-back state of the device from call to call, told
    apart by a number that the host counts up and a captured launch repeats:
    sort_pairs brings its own, zeroed in the stream."""
    text = open(os.path.join(REPO, "macmetalpy_b200", "csrc", "mmp_sort.cu")).read()
    body = text[text.index("int sort_pairs("):]
    body = body[:body.index("\n}\n")]
    assert "mmp_scan(" not in body and "scratch(" not in body
    scan = open(os.path.join(REPO, "macmetalpy_b200", "csrc", "mmp_scan.cu")).read()
    body = scan[scan.index("int scan_counts("):]
    body = body[:body.index("\n}\n")]
    assert "scan_state(" not in body
    grad = open(os.path.join(REPO, "macmetalpy_b200", "csrc", "mmp_embedding.cu")).read()
    assert "cudaMemsetAsync(zeroed, 0, state +" in grad
