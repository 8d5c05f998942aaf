#!/bin/bash
# A/B library: search_mfma.hip (or the file named in $FILE) built with the extra flags in $2 into tools/_ab/$1.so;
# run it through MI355RAG_LIB=tools/_ab/$1.so.  Flags and objects are those of the library itself (rag_amd/_build.py).
set -e
cd "$(dirname "$0")/.."
python -m rag_amd._build > /dev/null
mkdir -p tools/_ab
FILE=${FILE:-search_mfma}
/opt/rocm/bin/hipcc $(python -m rag_amd._build --flags $FILE.hip) $2 -c rag_amd/csrc/$FILE.hip -o tools/_ab/$1_$FILE.o
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o tools/_ab/$1.so $(python -m rag_amd._build --objects $FILE.hip) tools/_ab/$1_$FILE.o
echo built tools/_ab/$1.so
