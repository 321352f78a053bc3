"""In-tree build of the atomo_amd HIP extension for MI355X (gfx950).

    python setup.py build_ext --inplace

The .so lands at atomo_amd/ops/_atomo_hip*.so, beside its sources; it is
git-ignored.
"""

import os

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))

ext = CUDAExtension(
    name="atomo_amd.ops._atomo_hip",
    sources=[
        "atomo_amd/ops/csrc/bindings.cpp",
        "atomo_amd/ops/csrc/atomo_kernels.hip",
        "atomo_amd/ops/csrc/svd_batched.hip",
        "atomo_amd/ops/csrc/jacobi_eigh.hip",
        "atomo_amd/ops/csrc/linear_bindings.cpp",
        "atomo_amd/ops/csrc/linear_kernels.hip",
        "atomo_amd/ops/csrc/logit_bindings.cpp",
        "atomo_amd/ops/csrc/logit_kernels.hip",
    ],
    extra_compile_args={
        "cxx": ["-O3", "-std=c++17"],
        # no packed fp32 instructions: some of their forms have given wrong
        # results on this hardware
        "nvcc": ["-O3", "-std=c++17", "-Xclang", "-target-feature",
                 "-Xclang", "-packed-fp32-ops"],
    },
    libraries=["rocsolver", "rocblas"],
)

setup(
    name="atomo_amd",
    version="0.1.0",
    packages=["atomo_amd"],
    ext_modules=[ext],
    cmdclass={"build_ext": BuildExtension.with_options(no_python_abi_suffix=False)},
)
