"""CPU tests of the compiled kernels: hazards that the compiler does not see, because the
instruction that has to wait is written as inline assembly, and scratch memory."""
from __future__ import annotations

import kernel_code as K
from lsamp import _ffi


def test_scalar_addresses_of_loads_to_lds():
    """A vector instruction that writes a scalar register is five wait states ahead of a
    load that takes its address from there, on every path."""
    loads, stale = 0, []
    for f in K.functions(_ffi.LIB_PATH, "global_load_lds"):
        loads += sum(c.op.startswith("global_load_lds") for c in f.code)
        stale += [(f.name, f.code[i]) for i in K.stale_addresses(f)]
    assert loads > 1000, "the library's loads to LDS were not found"
    assert not stale, f"{len(stale)} loads, the first {stale[0]}"


def test_data_of_stores_past_the_caches():
    """A store's data is not overwritten by a vector instruction within two wait states."""
    for kernels, flags, least in (("k_norm", ("nt",), 50),
                                  ("k_resident", ("sc0", "sc1", "nt"), 6)):
        stores, unsettled = 0, []
        for f in K.functions(_ffi.LIB_PATH, "global_store_dwordx4", kernels):
            n, bad = K.unsettled_stores(f, flags)
            stores += n
            unsettled += [(f.name, f.code[i:i + 2]) for i in bad]
        assert stores >= least, f"{stores} stores of {kernels} were found"
        assert not unsettled, f"{len(unsettled)} stores, the first {unsettled[0]}"


def test_blocks_operators_use_no_scratch_memory():
    """8-bit products, norms and orthogonalised updates: no spills, and no called function
    whose state would lie there."""
    scratch = K.scratch_bytes(_ffi.LIB_PATH)
    ours = [k for k in scratch if any(part in k for part in (
        "k_gemmILi3E", "k_skinnyILi3E", "k_resident", "k_join_int8", "k_norm", "k_quantize",
        "BatchPlan", "k_start"))]
    assert len(ours) > 150
    assert not [(k, scratch[k]) for k in ours if scratch[k]]
