"""What a run cannot show: properties of the kernels' source that hold by the order of its statements."""
import os
import re

from conftest import PKG_DIR

CSRC = os.path.join(PKG_DIR, "csrc")


def source(name):
    """The file without its comments (positions of lines kept)."""
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def functions(text, pattern):
    """(name, body) of each device function whose body matches."""
    for m in re.finditer(r"MBP_DEV \w+ (\w+)\([^;{]*\) \{\n(.*?)\n\}", text, flags=re.S):
        if re.search(pattern, m.group(2)):
            yield m.group(1), m.group(2)


def test_warp_collective_tmem_accesses_reconverge_first():
    """tcgen05.ld / st / alloc / dealloc are .sync.aligned: a warp that comes from per-lane branches meets itself first."""
    found = 0
    for name, body in functions(source("tc.cuh"), r"tcgen05\.(ld|st)\.sync\.aligned"):
        before = body[:re.search(r"tcgen05\.(ld|st)\.sync\.aligned", body).start()]
        assert "__syncwarp();" in before, name
        found += 1
    assert found == 3
    for f in ("gemm.cu", "expert_gemm.cu"):
        text = source(f)
        for m in re.finditer(r"tcgen05\.(alloc|dealloc)\.", text):
            block = text[text.rindex("if (warp == 1) {", 0, m.start()):m.start()]
            assert "__syncwarp();" in block, (f, m.group(0))
        assert not re.search(r"tcgen05\.(ld|st)\.", text)  # only through the helpers


def test_escape_masks_in_front_of_matrix_instructions():
    """take_mask branches per lane; ldmatrix and mma.sync (.sync.aligned) follow it in the expert GEMV, tcgen05.st behind
    tc_st_a's own __syncwarp in the tensor-core kernels."""
    assert re.search(r"take_mask\([^;]*\);\s*__syncwarp\(\);", source("expert_gemv.cu"))


def test_decoded_tiles_are_stored_behind_a_fence():
    """tcgen05.st into a stage that earlier matrix products read: the wait for their commit orders the threads, and
    tcgen05.fence::after_thread_sync orders the store behind that wait."""
    for f in ("gemm.cu", "expert_gemm.cu"):
        text = source(f)
        stores = [m.start() for m in re.finditer(r"tc_st_a<", text)]
        assert stores
        for at in stores:
            wait = [m.end() for m in re.finditer(r"(mbar|warp)_wait\(oempty", text[:at])][-1]
            assert "tc_fence_after();" in text[wait:at], f


def test_copies_and_matrix_products_end_before_their_block():
    """A producer whose consumers gave up leaves copies on their way into the block's shared memory: every producer waits
    for its own, and every issuer for its products, under a limit of their own."""
    for f, rings in (("gemm.cu", 2), ("expert_gemv.cu", 1), ("expert_gemm.cu", 2)):
        text = source(f)
        assert len(re.findall(r"\bdrain_ring\(", text)) == rings, f
        if "tc_mma_ts(" in text:
            assert re.search(r"tc_commit\(done\);\s*mbar_wait\(done, 0, \w+, kDefaultWaitLimitNs\);", text), f
    # the GEMV waits where one of its two loops gives up
    assert len(re.findall(r"mbar_wait\([^{]*\{\s*await_copies\(full0,[^}]*break;", source("gemv.cu"))) == 2
    assert "kDefaultWaitLimitNs" in dict(functions(source("common.cuh"), "mbar_wait"))["drain_ring"]
