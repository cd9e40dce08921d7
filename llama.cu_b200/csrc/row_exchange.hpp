// How the CTAs of a cluster exchange one value each per row, and how they leave: the order of steps alone, for host and device.  What a step does on
// the machine is the port's (the softmax's in verify.cu).
//
// For each of two turns a CTA has a slot per CTA of the cluster and a barrier that ends when a value has come from each.  A row's values go into
// everyone's slots of its turn.  A CTA sends for a row only when it has all values of the rows before, so whoever waits for row r can be
// sent nothing of row r + 2, which has the same slots: the sender would need this CTA's value of row r + 1.
//
// Waits are bounded.  A CTA one of whose waits has run out sends nothing from then on: its threads' exchanges fail at once, so what it sent is
// always whole rows in a row, the argument above stands for those that still wait, and they run into limits of their own.
//
// Leaving.  A CTA that has had every value of its last row was sent everything it ever will be: it may go.  One that has given up may still be sent
// to: it stays until everyone else has gone or has given up too (neither sends), then until what they sent has landed.
#pragma once
#include <stdint.h>

#ifndef LCU_HD
#ifdef __CUDACC__
#define LCU_HD __host__ __device__
#else
#define LCU_HD
#endif
#endif

namespace lcu {

// One per thread; all threads of a CTA take the same steps.  Ahead of each exchange lies a barrier of the CTA, behind whatever else may give up.  Port:
//   started()     everyone's barriers are set up: waited for once
//   send(turn)    this thread's share of the row's value to everyone, and of the CTA's barrier's count
//   wait(turn, parity)  whether all values are there; bounded
//   gave_up(), give_up()  a flag of the CTA
//   together()    a barrier of the CTA
//   others()      until every CTA of the cluster has gone or is here
//   landed()      until no store to this CTA can be on its way
struct RowExchange {
    uint32_t row = 0;  // of the CTA's own, from 0 on

    LCU_HD uint32_t turn() const { return row & 1u; }
    LCU_HD uint32_t parity() const { return row >> 1 & 1u; }  // of the turn's barrier: it ends once every two rows
    template <class Port> LCU_HD bool exchange(Port &port) {
        if (row == 0) port.started();
        if (port.gave_up()) return false;
        port.send(turn());
        if (port.wait(turn(), parity())) return true;
        port.give_up();
        return false;
    }
    LCU_HD void next_row() { ++row; }
    template <class Port> LCU_HD void leave(Port &port) {  // behind one row or more
        port.together();  // no thread waits any more: all see the same flag
        if (!port.gave_up()) return;
        port.others();
        port.landed();
    }
};

}  // namespace lcu
