#!/bin/bash
# measurement aid: registers / scratch / occupancy of every kernel of a translation unit (compiler remarks, no GPU needed): tools/kres.sh [libfmarl | fmarl_memory | fmarl_block | fmarl_actions]
# compiled as __graft_entry__.build() does
U=${1:-libfmarl}
cd "$(dirname "$0")/.." && FLAGS=$(python3 -c "import sys, __graft_entry__ as g; print(*g.flags(sys.argv[1]))" $U) || exit 1
cd fair_marl_amd/csrc && ${HIPCC:-/opt/rocm/bin/hipcc} $FLAGS -Rpass-analysis=kernel-resource-usage -o /tmp/kres_lib.o $U.hip 2>&1 | python3 -c "
import sys,re
cur=None
for l in sys.stdin:
    m=re.search(r'Function Name: (\S+)',l)
    if m: cur=m.group(1); vals={}
    for k in ('VGPRs','ScratchSize \[bytes/lane\]','Occupancy \[waves/SIMD\]','SGPRs Spill'):
        m=re.search(r'    '+k+r': (\d+)',l)
        if m and cur: vals[k]=m.group(1)
    if cur and 'SGPRs Spill' in l and ' Spill: ' in l and 'VGPRs Spill' not in l:
        print('%-90s vgpr %4s scratch %4s occ %s' % (cur[:90], vals.get('VGPRs'), vals.get('ScratchSize \\\\[bytes/lane\\\\]'), vals.get('Occupancy \\\\[waves/SIMD\\\\]')))
"
