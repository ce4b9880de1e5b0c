"""mpserve_amd: MPServe's FP8 + Huffman-sidecar weight path on AMD MI355X (gfx950).

* ``mpserve_amd.mpserve_cuda`` — the reference's ``MPServe_cuda`` op surface
  (build + decode), over hand-written HIP kernels in ``libmpserve_amd.so``.
* ``mpserve_amd.decode.DecodePlan`` — one launch for many tensors.
* ``mpserve_amd.vllm_fp8_huffman`` — the vLLM ``fp8_huffman`` quantization method.
* ``mpserve_amd.mxfp4`` — 4-bit floating-point weights: quantization and products.
* ``mpserve_amd.int4`` — products with int4 weights, of an AWQ checkpoint or the AWQ decode ops.
* ``mpserve_amd.experts`` — a mixture's router and its balance loss, tokens to their experts and back,
  and products with MXFP4 and int4 experts;
  ``mpserve_amd.mxfp4_experts`` is a block of them.
"""
__version__ = "0.1.0"
