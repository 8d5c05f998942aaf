#!/bin/bash
# Builds the cycle-stamp debug library of the scan (tools/_trace/libtrace.so): search_mfma.hip with -DMF_TRACE
# and encoder.hip with -DFF_TRACE (extra flags in $1, e.g. -DMF_TRACE_U0=300), the other objects as built by rag_amd/_build.py,
# which also gives the flags.
set -e
cd "$(dirname "$0")/.."
python -m rag_amd._build > /dev/null
mkdir -p tools/_trace
/opt/rocm/bin/hipcc $(python -m rag_amd._build --flags search_mfma.hip) -DMF_TRACE $1 -c rag_amd/csrc/search_mfma.hip -o tools/_trace/search_mfma.o
/opt/rocm/bin/hipcc $(python -m rag_amd._build --flags encoder.hip) -DFF_TRACE $1 -c rag_amd/csrc/encoder.hip -o tools/_trace/encoder.o
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o tools/_trace/libtrace.so $(python -m rag_amd._build --objects search_mfma.hip encoder.hip) tools/_trace/encoder.o tools/_trace/search_mfma.o
echo built tools/_trace/libtrace.so
