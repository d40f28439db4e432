"""The encoder's kernels keep to their registers: no scratch and no spills in any variant (CPU only)."""
from test_build_guards import code_objects, kernel_resources, pytestmark  # noqa: F401

KERNELS = ("embed_kernel", "bucket_ids_kernel", "sort_ids_kernel", "embed_grad_kernel", "join_long_kernel",
           "embed_grad_few_kernel", "norm_kernel", "norm_grad_kernel", "norm_join_kernel", "adamw_kernel",
           "adam_values_kernel", "quantize_kernel", "matmul_kernel", "join_products_kernel", "matmul_few_kernel")


def test_no_scratch_in_the_encoders_kernels(code_objects):  # noqa: F811
    res = kernel_resources(code_objects)
    for name in KERNELS:
        # a kernel's mangled name holds its name's length before it
        found = {k: r for k, r in res.items() if f"{len(name)}{name}" in k}
        assert found, name
        for k, r in found.items():
            assert r["private_segment_fixed_size"] == 0 and r["vgpr_spill_count"] == 0, (k, r)
