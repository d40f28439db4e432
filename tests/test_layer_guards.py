"""The transformer layer's kernels keep to their registers: no scratch and no spills in any variant (CPU only)."""
from test_build_guards import code_objects, kernel_resources, pytestmark  # noqa: F401

KERNELS = ("rotary_kernel", "attention_kernel", "attention_dq_kernel", "attention_dkv_kernel", "attention_join_kernel",
           "product_kernel", "join_product_kernel", "slope_kernel", "pack_kernel", "few_kernel")


def test_no_scratch_in_the_layers_kernels(code_objects):  # noqa: F811
    res = kernel_resources(code_objects)
    for name in KERNELS:
        found = {k: r for k, r in res.items() if f"{len(name)}{name}" in k}
        assert found, name
        for k, r in found.items():
            assert r["private_segment_fixed_size"] == 0 and r["vgpr_spill_count"] == 0, (k, r)
